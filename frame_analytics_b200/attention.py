"""Attention operands: the norm of query and key heads with the rotation by
position, in one pass (no counterpart in the reference; ``csrc/qk_rotary.cu``).

A network trained against the package's losses normalises its queries and keys
so that attention logits stay bounded under orthogonalised updates
(:class:`frame_analytics_b200.Muon`), and rotates them by token position.
"""

from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import backend
from .functional import _reject_double_backward

__all__ = ["qk_norm_rotary"]

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_MAX_DIM = 512


# struct fa_heads and struct fa_qk_params of include/fa_b200.h as bytes: a call
# on one token takes a few microseconds on the GPU, so the host side counts
_HEADS = struct.Struct("@Pii3q").pack
_PARAMS = struct.Struct("@10i3P2q2Pd").pack


def _heads(t: torch.Tensor) -> bytes:
    b, l, h, _ = t.stride()
    return _HEADS(t.data_ptr(), t.shape[2], 0, b, l, h)


def _params(q, cos, sin, q_weight, k_weight, eps, positions, interleaved) -> bytes:
    code = backend.DTYPE_CODE[q.dtype]
    w = q_weight if q_weight is not None else k_weight
    if w is None:
        w_code, per_head = code, 0
    else:
        w_code, per_head = backend.DTYPE_CODE[w.dtype], w.dim() == 2
    b, l, _, d = q.shape
    rotary = table = cp = sp = pp = wide = pos_b = pos_l = 0
    if cos is not None:
        table, rotary = cos.shape
        rotary *= 2
        cp, sp = cos.data_ptr(), sin.data_ptr()
    if positions is not None:
        pp, wide = positions.data_ptr(), positions.dtype == torch.int64
        stride = positions.stride()
        pos_l = stride[-1]
        pos_b = stride[0] if len(stride) == 2 else 0
    return _PARAMS(code, w_code, b, l, d, rotary, interleaved, per_head, table, wide, cp, sp, pp,
                   pos_b, pos_l, 0 if q_weight is None else q_weight.data_ptr(),
                   0 if k_weight is None else k_weight.data_ptr(), eps)


def _forward(q, k, q_out, k_out, *rest):
    backend._call(q, backend.lib().fa_b200_qk_norm_rotary, _heads(q), _heads(k), _heads(q_out),
                  _heads(k_out), _params(q, *rest), backend._dev(q), backend._stream(q))


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, eps, positions, interleaved):
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        _forward(q, k, q_out, k_out, cos, sin, q_weight, k_weight, eps, positions, interleaved)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return q_out, k_out

    @staticmethod
    def backward(ctx, gq, gk):
        _reject_double_backward()
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        p = _params(q, cos, sin, q_weight, k_weight, ctx.eps, positions, ctx.interleaved)
        gq = gq if gq.stride(-1) == 1 else gq.contiguous()
        gk = gk if gk.stride(-1) == 1 else gk.contiguous()
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        need = ctx.needs_input_grad
        dqw = torch.empty_like(q_weight) if q_weight is not None and need[2] else None
        dkw = torch.empty_like(k_weight) if k_weight is not None and need[3] else None
        L = backend.lib()
        nb = backend._cached_ws("qk", L.fa_b200_qk_norm_rotary_backward_workspace_bytes,
                                q.shape[0], q.shape[1], q.shape[2], k.shape[2], q.shape[3])
        ws = backend.workspace(q, nb)
        backend._call(q, L.fa_b200_qk_norm_rotary_backward, _heads(q), _heads(k), _heads(gq),
                      _heads(gk), _heads(dq), _heads(dk), p, backend._ptr(dqw),
                      backend._ptr(dkw), ws.data_ptr(), ws.numel(), backend._dev(q), backend._stream(q))
        return dq, dk, dqw, dkw, None, None, None, None, None


def _check_weight(name, w, x, other):
    if w is None:
        return
    if w.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{name} must be {x.dtype} or float32, got {w.dtype}")
    if tuple(w.shape) not in ((x.shape[3],), (x.shape[2], x.shape[3])):
        raise ValueError(f"{name} must have shape ({x.shape[3]},) or "
                         f"({x.shape[2]}, {x.shape[3]}), got {tuple(w.shape)}")
    if other is not None and (other.dtype != w.dtype or other.dim() != w.dim()):
        raise ValueError("q_weight and k_weight must have one dtype and one number of dimensions")


def _check_out(name, o, x):
    if not torch.is_tensor(o) or o.shape != x.shape or o.dtype != x.dtype or o.device != x.device:
        raise ValueError(f"{name} must be a {x.dtype} tensor of shape {tuple(x.shape)} on {x.device}")
    if o.stride(-1) != 1 and o.shape[-1] != 1:
        raise ValueError(f"{name} must have unit stride in its last dimension")
    if any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
        raise ValueError(f"{name} has elements that share memory")


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _check_places(q_out, k_out, q, k) -> None:
    """Outputs start apart from one another and from every input but their own,
    which they then cover element for element.  (Overlaps that start elsewhere
    are the caller's to avoid.)"""
    po, pk = q_out.data_ptr(), k_out.data_ptr()
    for name, bad in (("out[0] and out[1]", po == pk),
                      ("out[0] and k", po == k.data_ptr()),
                      ("out[1] and q", pk == q.data_ptr()),
                      ("out[0] and q", po == q.data_ptr() and not _same_place(q_out, q)),
                      ("out[1] and k", pk == k.data_ptr() and not _same_place(k_out, k))):
        if bad:
            raise ValueError(f"{name} share memory")


def _reject_tangents(*tensors) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("qk_norm_rotary has no forward-mode derivative")


# Shapes and dtypes that passed _check: metadata, no tensor is kept.
_checked: set = set()


def _check(q, k, cos, sin, q_weight, k_weight, eps, positions) -> None:
    for name, t in (("q", q), ("k", k)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be (B, L, heads, D), got shape {tuple(t.shape)}")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be float16, bfloat16 or float32, got {t.dtype}")
    if q.dtype != k.dtype or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} differ in "
                         "batch, length, head size or dtype")
    dim = q.shape[3]
    if dim > _MAX_DIM or dim < 1:
        raise ValueError(f"the head size must be 1..{_MAX_DIM}, got {dim}")
    if q.shape[2] < 1 or k.shape[2] < 1:
        raise ValueError("q and k need at least one head each")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 \
                or sin.dtype != torch.float32:
            raise ValueError("cos and sin must be float32 tables of one shape (P, R/2)")
        if not 2 <= 2 * cos.shape[1] <= dim:
            raise ValueError(f"the tables rotate {2 * cos.shape[1]} of {dim} components")
    if positions is not None:
        if cos is None:
            raise ValueError("positions need cos and sin")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if tuple(positions.shape) not in ((q.shape[1],), (q.shape[0], q.shape[1])):
            raise ValueError(f"positions must be ({q.shape[1]},) or ({q.shape[0]}, {q.shape[1]}), "
                             f"got {tuple(positions.shape)}")
    elif cos is not None and q.shape[1] > cos.shape[0]:
        raise ValueError(f"{q.shape[1]} tokens for tables of {cos.shape[0]} positions")
    if not (eps >= 0.0):
        raise ValueError(f"eps must not be negative, got {eps}")
    _check_weight("q_weight", q_weight, q, k_weight)
    _check_weight("k_weight", k_weight, k, q_weight)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, cos: Optional[torch.Tensor] = None,
                   sin: Optional[torch.Tensor] = None, *,
                   q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                   out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalise every query and key head and rotate it by its token's position:
    ``y = R_p (w * x / sqrt(mean(x**2) + eps))``.  Differentiable once, in
    reverse mode, in the operands and the weights; ``cos`` and ``sin`` that want
    a gradient are refused.

    ``q`` (B, L, Hq, D) and ``k`` (B, L, Hk, D), float16 / bfloat16 / float32,
    may be views of a packed projection (any strides with unit stride in D; D
    at most 512).  ``cos`` / ``sin``: float32 (P, R/2) tables; the first
    ``R <= D`` components turn, in pairs (i, i + R/2), or (2i, 2i + 1) with
    ``interleaved``.  ``positions``: int32 / int64 (L,) or (B, L) rows of the
    tables, by default 0..L-1; a position outside the tables gives NaN for its
    token (and then for the weights' gradients).  Weights: (D,) shared by the
    heads, or (heads, D); in the operands' dtype or float32.

    Returns contiguous (B, L, Hq, D) and (B, L, Hk, D).  ``out=(q_out, k_out)``
    writes there instead (any strides with unit stride in D: a slice of a cache,
    or the inputs themselves, and no other memory that the call reads or
    writes); it takes no part in autograd."""
    eps = float(eps)
    key = (q.shape, q.dtype, k.shape, k.dtype, eps, *[
        None if t is None else (t.shape, t.dtype)
        for t in (cos, sin, positions, q_weight, k_weight)])
    if key not in _checked:
        _check(q, k, cos, sin, q_weight, k_weight, eps, positions)
        if len(_checked) > 4096:
            _checked.clear()
        _checked.add(key)
    tracked = torch.is_grad_enabled()
    if tracked and cos is not None and (cos.requires_grad or sin.requires_grad):
        raise ValueError("qk_norm_rotary gives cos and sin no gradient: detach them")
    if forward_ad._current_level >= 0:
        _reject_tangents(q, k, cos, sin, q_weight, k_weight)
    index = q.get_device()
    for t in (q, k, cos, sin, q_weight, k_weight, positions):
        if t is not None and t.get_device() != index or index < 0:
            backend.require_cuda(*[u for u in (q, k, cos, sin, q_weight, k_weight, positions)
                                   if u is not None])
            raise ValueError("all tensors must be on one device")
    grad = tracked and any(
        t is not None and t.requires_grad for t in (q, k, q_weight, k_weight))
    if out is not None:
        if grad:
            raise ValueError("out= takes no part in autograd; call under torch.no_grad()")
        if not isinstance(out, (tuple, list)) or len(out) != 2:
            raise ValueError("out must be a pair (q_out, k_out)")
        _check_out("out[0]", out[0], q)
        _check_out("out[1]", out[1], k)
    q = q if q.stride(-1) == 1 else q.contiguous()
    k = k if k.stride(-1) == 1 else k.contiguous()
    if cos is not None:
        cos, sin = cos.contiguous(), sin.contiguous()
    q_weight = None if q_weight is None else q_weight.contiguous()
    k_weight = None if k_weight is None else k_weight.contiguous()
    rest = (cos, sin, q_weight, k_weight, eps, positions, bool(interleaved))
    if q.shape[0] == 0 or q.shape[1] == 0:
        if out is not None:
            return out[0], out[1]
        # connected to the graph, so that a backward gives zero gradients
        zero = sum(w.sum() * 0 for w in (q_weight, k_weight) if w is not None)
        return ((q * 1.0 + zero).to(q.dtype).contiguous(),
                (k * 1.0 + zero).to(k.dtype).contiguous())
    if grad:
        return _QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, eps, positions,
                                   bool(interleaved))
    if out is None:
        out = (torch.empty(q.shape, dtype=q.dtype, device=q.device),
               torch.empty(k.shape, dtype=k.dtype, device=k.device))
        _forward(q, k, out[0], out[1], *rest)
    else:
        _check_places(out[0], out[1], q, k)
        _forward(q, k, out[0], out[1], *rest)
        torch.autograd.graph.increment_version(out)
    return out[0], out[1]
