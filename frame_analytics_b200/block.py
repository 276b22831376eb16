"""A transformer block's norm, activation and products with what they keep for the
backward pass in 8 bits (no counterpart in the reference; ``csrc/keep8.cu``,
``csrc/layer_norm.cu``, ``csrc/linear8.cu``).

A network that restores whole frames keeps the input of every norm, activation
and product until its gradient comes back; these inputs, not the weights, fill
the memory.  ``pack8`` holds them in 68 bytes (float32: 72) for every 64 values of
a row, also where the last 64 are not all there: long rows take 1.06 (1.13) bytes a
value, and only rows of up to 34, or 65 to 68, 16-bit (18 float32) values no less
than they do themselves.  ``layer_norm``, ``gelu8`` and ``linear8`` read that form in
their backward passes without unpacking it first.
"""

from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import backend
from .functional import _reject_double_backward

__all__ = ["Packed8", "pack8", "unpack8", "layer_norm", "gelu8", "linear8"]

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_GROUP = 64
_MAX_WIDTH = 1 << 24
_MAX_SIDE, _MAX_ROWS = (1 << 22) - 64, 1 << 27  # of a product
# struct fa_norm of include/fa_b200.h as bytes
_NORM = struct.Struct("@2iq2idPqPq5P").pack
# struct fa_linear8
_LINEAR = struct.Struct("@4iqPqPqPq7P").pack


class Packed8(NamedTuple):
    """A tensor in 8 bits, made by :func:`pack8`.

    ``codes``: uint8 (..., 64 G), G groups of 64 along the last dimension, zeros
    past its end.  ``ranges``: each group's lowest value and step, int32 (..., G)
    for 16-bit tensors (the lowest value in the low half, the step as bfloat16 in
    the high half), float32 (..., G, 2) for float32.  ``shape`` and ``dtype`` are
    the tensor's own."""

    codes: torch.Tensor
    ranges: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype


def _check_values(name: str, x: torch.Tensor, most: int) -> None:
    if not torch.is_tensor(x):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= most:
        raise ValueError(f"{name} must have a last dimension of 1..{most}, got shape "
                         f"{tuple(x.shape)}")


def _on_one_device(x: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    index = x.get_device()
    for t in (x, *others):
        if t is not None and (t.get_device() != index or index < 0):
            backend.require_cuda(*[u for u in (x, *others) if u is not None])
            raise ValueError("all tensors must be on one device")


def _reject_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """As a matrix of rows with unit stride; a copy where that takes one."""
    width = t.shape[-1]
    if t.is_neg():  # an imaginary part, or its gradient: the sign is not in memory
        t = t.resolve_neg()
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1):
        return t
    if t.stride(-1) != 1 and width > 1:
        t = t.contiguous()
    return t.reshape(-1, width)


def _packed_like(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    lead, groups = x.shape[:-1], -(-x.shape[-1] // _GROUP)
    codes = torch.empty((*lead, groups * _GROUP), dtype=torch.uint8, device=x.device)
    if x.dtype == torch.float32:
        return codes, torch.empty((*lead, groups, 2), dtype=torch.float32, device=x.device)
    return codes, torch.empty((*lead, groups), dtype=torch.int32, device=x.device)


def _kept_like(x: torch.Tensor, rows: int, stats: bool) -> Tuple[torch.Tensor, int, int]:
    """One buffer for the codes, two floats a row (``stats``) and the ranges, in this
    order; the offsets of the latter two.  An allocation costs as much host time as a
    launch."""
    groups = -(-x.shape[-1] // _GROUP)
    at = rows * groups * _GROUP
    ranges = at + (8 * rows if stats else 0)
    size = ranges + rows * groups * (8 if x.dtype == torch.float32 else 4)
    return torch.empty(size, dtype=torch.uint8, device=x.device), at, ranges


def _empty(like: torch.Tensor) -> torch.Tensor:
    """Contiguous, of the same shape."""
    if like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty(like.shape, dtype=like.dtype, device=like.device)


# --------------------------------------------------------------------------- #
# packing
# --------------------------------------------------------------------------- #

def _pack_into(x: torch.Tensor, codes: int, ranges: int) -> None:
    r = _rows(x)
    backend._call(r, backend.lib().fa_b200_pack8, r.data_ptr(), r.stride(0),
                  backend.DTYPE_CODE[x.dtype], r.shape[0], r.shape[1], codes, ranges,
                  backend._dev(r), backend._stream(r))


def _pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    codes, ranges = _packed_like(x)
    if x.numel():
        _pack_into(x, codes.data_ptr(), ranges.data_ptr())
    return codes, ranges


def pack8(x: torch.Tensor) -> Packed8:
    """A tensor (float16, bfloat16 or float32, any strides) in 8 bits.

    Groups of 64 values of the last dimension (the last group may be short) hold
    their lowest value ``lo``, a step ``s`` (the smallest power of two, from
    2^-126 up, with ``max - lo <= 255 s``) and codes ``rint((x - lo) / s)`` of 8
    bits.  A value comes back as ``code s + lo``, at most ``(max - lo) / 255`` off
    (before it is rounded to the dtype).  A group that holds an infinity or a NaN,
    or whose spread is past float32's range, comes back as NaNs.  Takes no part
    in autograd."""
    _check_values("x", x, 2 ** 31 - 1)
    backend.require_cuda(x)
    return Packed8(*_pack(x.detach()), x.shape, x.dtype)


def _check_packed(p: Packed8) -> None:
    if not isinstance(p, Packed8):
        raise TypeError(f"unpack8 takes what pack8 returns, got {type(p).__name__}")
    if p.dtype not in _DTYPES or len(p.shape) < 1 or p.shape[-1] < 1:
        raise ValueError(f"no packed tensor of shape {tuple(p.shape)} and {p.dtype}")
    lead, groups = tuple(p.shape[:-1]), -(-p.shape[-1] // _GROUP)
    wide = p.dtype == torch.float32
    for name, t, shape, dtype in (
            ("codes", p.codes, (*lead, groups * _GROUP), torch.uint8),
            ("ranges", p.ranges, (*lead, groups, 2) if wide else (*lead, groups),
             torch.float32 if wide else torch.int32)):
        if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dtype} of shape {shape}, got {t.dtype} "
                             f"{tuple(t.shape)}")


def unpack8(p: Packed8) -> torch.Tensor:
    """The values that a packed tensor stands for, contiguous, in its dtype."""
    _check_packed(p)
    codes, ranges = p.codes.detach(), p.ranges.detach()
    _on_one_device(codes, ranges)
    out = torch.empty(tuple(p.shape), dtype=p.dtype, device=codes.device)
    if out.numel():
        # a buffer that was moved may start anywhere
        codes = codes if codes.data_ptr() % 16 == 0 else codes.clone()
        ranges = ranges if ranges.data_ptr() % 8 == 0 else ranges.clone()
        width = p.shape[-1]
        backend._call(out, backend.lib().fa_b200_unpack8, codes.data_ptr(), ranges.data_ptr(),
                      backend.DTYPE_CODE[p.dtype], out.numel() // width, width, out.data_ptr(),
                      width, backend._dev(out), backend._stream(out))
    return out


# --------------------------------------------------------------------------- #
# layer norm
# --------------------------------------------------------------------------- #

def _norm_params(x, residual, weight, bias, eps, stats, codes, ranges, rows, width, dtype) -> bytes:
    """`x` and `residual`: rows; `stats`, `codes` and `ranges`: addresses."""
    w = weight if weight is not None else bias
    code = backend.DTYPE_CODE[dtype]
    return _NORM(code, code if w is None else backend.DTYPE_CODE[w.dtype], rows, width, 0, eps,
                 0 if x is None else x.data_ptr(), width if x is None else x.stride(0),
                 0 if residual is None else residual.data_ptr(),
                 0 if residual is None else residual.stride(0),
                 0 if weight is None else weight.data_ptr(),
                 0 if bias is None else bias.data_ptr(), stats, codes, ranges)


def _norm_forward(x, residual, weight, bias, eps, stats, codes, ranges):
    y = _empty(x)
    total = None if residual is None else torch.empty_like(y)
    xr, rr = _rows(x), None if residual is None else _rows(residual)
    p = _norm_params(xr, rr, weight, bias, eps, stats, codes, ranges, *xr.shape, x.dtype)
    backend._call(y, backend.lib().fa_b200_layer_norm, p, y.data_ptr(), backend._ptr(total),
                  backend._dev(y), backend._stream(y))
    return y, total


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, keep8):
        ctx.set_materialize_grads(False)
        rows = x.numel() // x.shape[-1]
        if keep8:
            kept, stats, ranges = _kept_like(x, rows, True)
            at = kept.data_ptr()
            y, total = _norm_forward(x, residual, weight, bias, eps, at + stats, at, at + ranges)
            ctx.save_for_backward(kept, None, weight, bias)
            ctx.at = (stats, ranges)
        else:
            stats = torch.empty(2 * rows, dtype=torch.float32, device=x.device)
            y, total = _norm_forward(x, residual, weight, bias, eps, stats.data_ptr(), 0, 0)
            ctx.save_for_backward(stats, x if residual is None else total, weight, bias)
            ctx.at = None
        ctx.eps = eps
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx, gy, gsum=None):
        _reject_double_backward()
        need = ctx.needs_input_grad
        if gy is None:  # the norm itself took no part
            return (gsum if need[0] else None, gsum if need[1] else None, None, None, None, None)
        kept, s, weight, bias = ctx.saved_tensors
        dx = _empty(gy)
        dw = torch.empty_like(weight) if weight is not None and need[2] else None
        db = torch.empty_like(bias) if bias is not None and need[3] else None
        g, gs = _rows(gy), None if gsum is None else _rows(gsum)
        rows, width = g.shape
        L = backend.lib()
        ws, size = None, 0
        if dw is not None or db is not None:
            size = backend._cached_ws("norm", L.fa_b200_layer_norm_backward_workspace_bytes,
                                      rows, width, backend._dev(g))
            ws = torch.empty(size, dtype=torch.uint8, device=g.device)
        at = kept.data_ptr()
        if ctx.at is None:
            s = _rows(s)
            p = _norm_params(s, None, weight, bias, ctx.eps, at, 0, 0, rows, width, g.dtype)
        else:
            p = _norm_params(None, None, weight, bias, ctx.eps, at + ctx.at[0], at, at + ctx.at[1],
                             rows, width, g.dtype)
        backend._call(g, L.fa_b200_layer_norm_backward, p, g.data_ptr(), g.stride(0),
                      backend._ptr(gs), 0 if gs is None else gs.stride(0), dx.data_ptr(),
                      backend._ptr(dw), backend._ptr(db), backend._ptr(ws), size, backend._dev(g),
                      backend._stream(g))
        return dx if need[0] else None, dx if need[1] else None, dw, db, None, None


def _check_affine(name: str, w: Optional[torch.Tensor], x: torch.Tensor) -> None:
    if w is None:
        return
    if not torch.is_tensor(w):
        raise TypeError(f"{name} must be a tensor or None, got {type(w).__name__}")
    if w.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{name} must be {x.dtype} or float32, got {w.dtype}")
    if tuple(w.shape) != (x.shape[-1],):
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(w.shape)}")


def _autocast_norm(x, residual, weight, bias):
    """Under autocast the norm's operands come in two types: products give its own, what
    they are added to and the weights may be in another.  Such operands meet in float32."""
    def ours(*tensors):
        return all(t is None or torch.is_tensor(t) and t.dtype in _DTYPES for t in tensors)

    if ours(x, residual) and residual is not None and x.dtype != residual.dtype:
        x, residual = x.float(), residual.float()
    types = {t.dtype for t in (weight, bias) if torch.is_tensor(t)}
    if ours(x, weight, bias) and not types <= {x.dtype} and types != {torch.float32}:
        weight, bias = (None if t is None else t.float() for t in (weight, bias))
    return x, residual, weight, bias


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *,
               residual: Optional[torch.Tensor] = None, eps: float = 1e-5, keep8: bool = False
               ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Layer norm over the last dimension, ``(x - mean) / sqrt(variance + eps) *
    weight + bias``; differentiable once, in reverse mode.

    With ``residual`` (``x``'s shape and dtype) the norm is that of ``s = x +
    residual``, rounded to the dtype, and the call returns ``(y, s)``: the block's
    residual sum costs no pass of its own, forward or backward.

    ``x`` (..., N): float16, bfloat16 or float32, any strides; N at most 2^24.
    ``weight`` and ``bias``, either or both: (N,), one dtype, ``x``'s or float32.
    Results are contiguous.  Mean, variance and the weights' gradients are
    summed in float32, in an order that does not change from run to run.  Under
    autocast ``x`` and ``residual`` of two dtypes are taken, and returned, as float32,
    and so are weights that do not fit.

    ``keep8``: keep ``x`` (or ``s``) for the backward pass as :func:`pack8` holds
    it, with the exact mean and deviation, instead of itself."""
    if torch.is_autocast_enabled("cuda"):
        x, residual, weight, bias = _autocast_norm(x, residual, weight, bias)
    _check_values("x", x, _MAX_WIDTH)
    if residual is not None and not torch.is_tensor(residual):
        raise TypeError(f"residual must be a tensor or None, got {type(residual).__name__}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {x.dtype} of shape {tuple(x.shape)}, got "
                         f"{residual.dtype} {tuple(residual.shape)}")
    _check_affine("weight", weight, x)
    _check_affine("bias", bias, x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one dtype")
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    _reject_tangents("layer_norm", x, residual, weight, bias)
    _on_one_device(x, residual, weight, bias)
    if weight is not None:
        weight = weight.resolve_neg().contiguous()
    if bias is not None:
        bias = bias.resolve_neg().contiguous()
    if x.numel() == 0:
        # connected to the graph, so that a backward gives zero gradients
        y = (x if residual is None else x + residual) * 1.0
        for w in (weight, bias):
            y = y if w is None else y + (w.sum() * 0).to(y.dtype)
        return y if residual is None else (y, x + residual)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        return _LayerNorm.apply(x, residual, weight, bias, eps, bool(keep8))
    y, total = _norm_forward(x, residual, weight, bias, eps, 0, 0, 0)
    return y if residual is None else (y, total)


# --------------------------------------------------------------------------- #
# activation
# --------------------------------------------------------------------------- #

def _gelu_forward(x, tanh_form, codes, ranges):
    y = _empty(x)
    r = _rows(x)
    backend._call(r, backend.lib().fa_b200_gelu8, r.data_ptr(), r.stride(0),
                  backend.DTYPE_CODE[x.dtype], r.shape[0], r.shape[1], tanh_form, y.data_ptr(),
                  codes, ranges, backend._dev(r), backend._stream(r))
    return y


class _Gelu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tanh_form):
        kept, ranges, _ = _kept_like(x, x.numel() // x.shape[-1], False)
        at = kept.data_ptr()
        y = _gelu_forward(x, tanh_form, at, at + ranges)
        ctx.save_for_backward(kept)
        ctx.ranges, ctx.tanh_form = ranges, tanh_form
        return y

    @staticmethod
    def backward(ctx, gy):
        _reject_double_backward()
        kept, = ctx.saved_tensors
        at = kept.data_ptr()
        dx = _empty(gy)
        g = _rows(gy)
        backend._call(g, backend.lib().fa_b200_gelu8_backward, g.data_ptr(), g.stride(0), at,
                      at + ctx.ranges, backend.DTYPE_CODE[gy.dtype], g.shape[0], g.shape[1],
                      ctx.tanh_form, dx.data_ptr(), backend._dev(g), backend._stream(g))
        return dx, None


def gelu8(x: torch.Tensor, *, approximate: str = "none") -> torch.Tensor:
    """``x Phi(x)``, or with ``approximate="tanh"`` ``x (1 + tanh(sqrt(2 / pi) (x +
    0.044715 x^3))) / 2``; the backward pass takes the slope at the values that
    :func:`pack8` keeps of ``x``, so ``x`` itself need not be kept.  Differentiable
    once, in reverse mode.

    ``x``: float16, bfloat16 or float32, any strides; the result is contiguous.
    The value is that of ``x`` itself."""
    _check_values("x", x, 2 ** 31 - 1)
    if approximate not in ("none", "tanh"):
        raise ValueError(f"approximate must be 'none' or 'tanh', got {approximate!r}")
    _reject_tangents("gelu8", x)
    backend.require_cuda(x)
    if x.numel() == 0:
        return x * 1.0
    tanh_form = int(approximate == "tanh")
    if torch.is_grad_enabled() and x.requires_grad:
        return _Gelu8.apply(x, tanh_form)
    return _gelu_forward(x, tanh_form, None, None)


# --------------------------------------------------------------------------- #
# products
# --------------------------------------------------------------------------- #

_linear_ws: dict = {}


def _linear_call(fn, t: torch.Tensor, rows: int, inputs: int, outputs: int, x, dy, weight, bias,
                 codes: int, ranges: int, y, dx, dw, db) -> None:
    """One of the two entries on `t`'s device; `x` and `dy` are rows, all but the
    addresses `codes` and `ranges` tensors or None."""
    at = [0 if v is None else v.data_ptr() for v in (x, dy, weight, bias, y, dx, dw, db)]
    p = _LINEAR(backend.DTYPE_CODE[t.dtype], inputs, outputs, 0, rows,
                at[0], 0 if x is None else x.stride(0), at[1], 0 if dy is None else dy.stride(0),
                at[2], 0 if weight is None else weight.stride(0), at[3], codes, ranges, *at[4:])
    device = backend._dev(t)
    # what the size depends on: the sizes, which results, and which operands are copied
    key = (p[:24], device, *[bool(v) for v in at[4:]], at[0] % 16, at[1] % 16, at[2] % 16,
           *[v is not None and v.stride(0) for v in (x, dy, weight)])
    size = _linear_ws.get(key)
    if size is None:
        size = backend._ws_query(backend.lib().fa_b200_linear8_workspace_bytes, p, device)
        if len(_linear_ws) > 4096:
            _linear_ws.clear()
        _linear_ws[key] = size
    ws = torch.empty(size, dtype=torch.uint8, device=t.device) if size else None
    backend._call(t, fn, p, backend._ptr(ws), size, device, backend._stream(t))


def _linear_forward(x, weight, bias, kept, ranges: int) -> torch.Tensor:
    """The product, and x packed into `kept` where that is given."""
    r = _rows(x)
    rows, inputs = r.shape
    outputs = weight.shape[0]
    fn = backend.lib().fa_b200_linear8
    at = 0 if kept is None else kept.data_ptr()
    if weight.stride(1) != 1 and inputs > 1:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.resolve_neg().contiguous()
    y = x.new_empty((*x.shape[:-1], outputs))
    _linear_call(fn, r, rows, inputs, outputs, r, None, weight, bias, at,
                 at + ranges if at else 0, y, None, None, None)
    return y


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        kept, ctx.ranges = None, 0
        if ctx.needs_input_grad[1]:
            kept, ctx.ranges, _ = _kept_like(x, x.numel() // x.shape[-1], False)
        y = _linear_forward(x, weight, bias, kept, ctx.ranges)
        ctx.save_for_backward(kept, weight)
        return y

    @staticmethod
    def backward(ctx, gy):
        _reject_double_backward()
        kept, weight = ctx.saved_tensors
        need, (outputs, inputs) = ctx.needs_input_grad, weight.shape
        g = _rows(gy)
        dx = dw = db = w = None
        at = 0
        if need[0]:
            dx = g.new_empty((*gy.shape[:-1], inputs))
            w = weight if weight.stride(1) == 1 or inputs == 1 else weight.contiguous()
        if need[1]:
            dw, at = g.new_empty((outputs, inputs)), kept.data_ptr()
        if need[2]:
            db = g.new_empty(outputs)
        _linear_call(backend.lib().fa_b200_linear8_backward, g, g.shape[0], inputs, outputs, None,
                     g, w, None, at, at + ctx.ranges if at else 0, None, dx, dw, db)
        return dx, dw, db


def linear8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None
            ) -> torch.Tensor:
    """``x W^T + bias`` that keeps ``x`` for the backward pass as :func:`pack8`
    holds it: the weight's gradient ``dy^T x`` takes ``x`` from the 8-bit form.
    Differentiable once, in reverse mode.

    ``x`` (..., K), ``weight`` (M, K), ``bias`` (M,): one dtype, float16, bfloat16
    or float32 (under autocast its dtype), any strides; K and M at most 4194240, and
    2^27 rows.  ``x`` is packed only where the weight wants a gradient.

    All products are this package's own, with float32 sums that are rounded once,
    however an axis is split: float16 and bfloat16 on the tensor cores, float32 in
    float32 (torch's settings for reduced precision do not matter)."""
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        if to in _DTYPES:
            x, weight, bias = (t.to(to) if torch.is_tensor(t) and t.dtype in _DTYPES else t
                               for t in (x, weight, bias))
    _check_values("x", x, _MAX_SIDE)
    if x.numel() // x.shape[-1] > _MAX_ROWS:
        raise ValueError(f"x of shape {tuple(x.shape)} has more than {_MAX_ROWS} rows")
    if not torch.is_tensor(weight) or weight.dim() != 2 or weight.shape[1] != x.shape[-1] \
            or weight.dtype != x.dtype:
        raise ValueError(f"weight must be {x.dtype} of shape (M, {x.shape[-1]}), got "
                         f"{getattr(weight, 'dtype', type(weight))} "
                         f"{tuple(getattr(weight, 'shape', ()))}")
    outputs = weight.shape[0]
    if not 1 <= outputs <= _MAX_SIDE:
        raise ValueError(f"the weight must have 1..{_MAX_SIDE} rows, got {outputs}")
    if bias is not None and not torch.is_tensor(bias):
        raise TypeError(f"bias must be a tensor or None, got {type(bias).__name__}")
    if bias is not None and (tuple(bias.shape) != (outputs,) or bias.dtype != x.dtype):
        raise ValueError(f"bias must be {x.dtype} of shape ({outputs},), got {bias.dtype} "
                         f"{tuple(bias.shape)}")
    _reject_tangents("linear8", x, weight, bias)
    _on_one_device(x, weight, bias)
    weight = weight.resolve_neg()
    if x.numel() == 0:
        return F.linear(x, weight, bias)
    if torch.is_grad_enabled() and (
            weight.requires_grad or x.requires_grad or bias is not None and bias.requires_grad):
        return _Linear8.apply(x, weight, bias)
    return _linear_forward(x, weight, bias, None, 0)
