"""Orthogonalised updates of weight matrices: the step from a loss's gradient to
new weights (no counterpart in the reference; ``csrc/orthogonalize.cu``).

``orthogonalize`` maps the singular values of a matrix towards 1 by
Newton-Schulz products; ``muon_step`` and the optimiser :class:`Muon` apply it
to momentum, in place, for a whole list of matrices at once.
"""

from __future__ import annotations

import ctypes
import math
import struct
from typing import Iterable, Optional, Sequence

import torch

from . import backend

__all__ = ["orthogonalize", "muon_step", "Muon", "NEWTON_SCHULZ"]

# The quintic whose five applications take every singular value in about
# [0.003, 1] to within about 0.3 of 1.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_MAX_STEPS = 32
_coef_cache: dict = {}
# struct fa_matrix of include/fa_b200.h as bytes
_MATRIX = struct.Struct("@3P2i2qd").pack


def _coefficients(coefficients, steps: int):
    """(ctypes array of steps x 3 doubles); one triple serves every step.
    Coefficients under which a singular value of 1 or less could leave the
    range of the kernels' number formats are refused."""
    if not isinstance(steps, int) or isinstance(steps, bool) or not 1 <= steps <= _MAX_STEPS:
        raise ValueError(f"steps must be a whole number 1..{_MAX_STEPS}, got {steps!r}")
    try:
        rows = tuple(tuple(float(v) for v in c) for c in coefficients) \
            if hasattr(coefficients[0], "__len__") else (tuple(float(v) for v in coefficients),) * steps
    except (TypeError, IndexError, ValueError):
        raise ValueError("coefficients must be a triple, or one triple for each step") from None
    key = (rows, steps)
    if key in _coef_cache:
        return _coef_cache[key]
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"coefficients must be a triple, or {steps} triples")
    if not all(math.isfinite(v) for r in rows for v in r):
        raise ValueError("coefficients must be finite")
    top = 1.0
    for a, b, c in rows:
        s = [top * 1.01 * i / 2048 for i in range(2049)]
        top = max(max(abs(v * (a + b * v * v + c * v ** 4)) for v in s), 1e-30)
        inner = max(abs(b * v * v + c * v ** 4) for v in s)
        if top > 64.0 or inner > 4096.0:
            raise ValueError(f"coefficients {(a, b, c)} let the iteration grow: singular values "
                             "that start at or below 1 must stay below 64")
    arr = (ctypes.c_double * (3 * steps))(*[v for r in rows for v in r])
    if len(_coef_cache) > 64:
        _coef_cache.clear()
    _coef_cache[key] = arr
    return arr


_MAX_SHORT, _MAX_LONG = 32768, 1 << 22


def _check_size(name: str, rows: int, cols: int) -> None:
    if min(rows, cols) > _MAX_SHORT or max(rows, cols) > _MAX_LONG:
        raise ValueError(f"{name} of {rows} x {cols}: the shorter side is at most {_MAX_SHORT}, "
                         f"the longer {_MAX_LONG}")


def _run(fn, mats, count: int, like: torch.Tensor, *args) -> None:
    L = backend.lib()
    code = backend.DTYPE_CODE[like.dtype]
    size = ctypes.c_size_t(0)
    backend._cabi.check(L.fa_b200_orthogonalize_workspace_bytes(mats, count, code,
                                                                ctypes.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=like.device)
    backend._call(like, fn, mats, count, code, *args, ws.data_ptr(), size.value,
                  backend._dev(like), backend._stream(like))


def orthogonalize(x: torch.Tensor, *, steps: int = 5,
                  coefficients: Sequence = NEWTON_SCHULZ) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of a matrix (m, n) or a stack (..., m, n):
    with ``X = x / |x|_F``, `steps` times ``X <- a X + (b A + c A^2) X``,
    ``A = X X^T`` (on the shorter side).  Every singular value s of X follows
    ``s (a + b s^2 + c s^4)``.

    float16, bfloat16 or float32 in and out; the result is contiguous.  bfloat16
    runs one tensor-core product per matrix product (about 1e-3 relative before
    the output is rounded); float16 and float32 run three (about 1e-6), and
    matrices up to 64 x 128 run in float32.  The shorter side is at most 32768,
    the longer 4194304.
    ``coefficients``: a triple (a, b, c), or one for each step.  A zero matrix
    gives zeros; one that holds an infinity or a NaN gives NaN.  The result
    takes no part in autograd."""
    if x.dim() < 2:
        raise ValueError(f"orthogonalize takes (..., m, n), got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"orthogonalize takes float16, bfloat16 or float32, got {x.dtype}")
    coef = _coefficients(coefficients, steps)
    m, n = x.shape[-2:]
    if x.numel():
        _check_size("a matrix", m, n)
    backend.require_cuda(x)
    x = x.detach()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return out
    x3 = x.reshape(-1, m, n)
    if (x3.stride(2) != 1 and n > 1) or (x3.stride(1) < n and m > 1):
        x3 = x3.contiguous()
    count, item = x3.shape[0], x.element_size()
    sb, sr = x3.stride(0) * item, x3.stride(1) if m > 1 else n
    src, dst = x3.data_ptr(), out.data_ptr()
    mats = b"".join([_MATRIX(src + i * sb, dst + i * m * n * item, 0, m, n, sr, n, 0.0)
                     for i in range(count)])
    _run(backend.lib().fa_b200_orthogonalize, mats, count, x, coef, steps)
    return out


def _rows_layout(w: torch.Tensor) -> Optional[torch.Tensor]:
    """`w` (2-D or more) as a contiguous matrix whose rows are its first
    dimension, or None.  A channels-last kernel keeps its own order of columns:
    permuting columns permutes those of the result."""
    if w.is_contiguous():
        return w.view(w.shape[0], -1)
    if w.dim() == 4 and w.is_contiguous(memory_format=torch.channels_last):
        return w.permute(0, 2, 3, 1).view(w.shape[0], -1)
    return None


def _like_layout(t: torch.Tensor, w: torch.Tensor) -> Optional[torch.Tensor]:
    """`t` as a matrix with `w`'s order of columns, without a copy, or None."""
    if t.stride() == w.stride() or (t.is_contiguous() and w.is_contiguous()):
        return _rows_layout(t)
    if not w.is_contiguous() and t.is_contiguous(memory_format=torch.channels_last):
        return t.permute(0, 2, 3, 1).view(t.shape[0], -1)
    return None


def _copied(t: torch.Tensor, like: torch.Tensor, name: str, back: list) -> torch.Tensor:
    """A copy of `t` with `like`'s order of elements, to be written back."""
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} has elements that share memory")
    c = torch.empty_like(like, dtype=t.dtype).copy_(t.detach())
    back.append((t.detach(), c))
    return c


_SCALES = ("aspect", "rms", "none")


def _scale(kind: str, rows: int, cols: int) -> float:
    if kind == "aspect":
        return math.sqrt(max(1.0, rows / cols))
    if kind == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    return 1.0


def muon_step(weights: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
              momenta: Sequence[torch.Tensor], *, lr: float, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, scale: str = "aspect",
              steps: int = 5, coefficients: Sequence = NEWTON_SCHULZ) -> None:
    """One optimiser step on a list of weight matrices, in place:

    ``M <- momentum M + G``;  ``U = G + momentum M`` (``nesterov``) or ``M``;
    ``W <- (1 - lr weight_decay) W - lr s orthogonalize(U)``.

    ``weights`` (float16, bfloat16 or float32, one dtype; two dimensions or
    more, rows = the first, the others flattened) and ``momenta`` (float32, the
    weights' shapes) are updated; ``grads`` have the weights' dtype.  ``scale``
    s: ``"aspect"`` sqrt(max(1, rows / cols)), ``"rms"`` 0.2 sqrt(max(rows,
    cols)), ``"none"`` 1.  Contiguous tensors and channels-last kernels are used
    where they lie, others through copies.

    One sequence of launches serves up to 128 matrices of up to 8 shapes, and 2
    GiB of workspace; longer lists take several.  Matrices up to 64 x 128 have
    launches of 128 of their own.  The momentum is float32 whatever the weights;
    the products are orthogonalize's for the weights' dtype, so larger bfloat16
    weights take an update that is about 1e-3 (relative) off, beside their own
    rounding."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    if not len(weights) == len(grads) == len(momenta):
        raise ValueError(f"{len(weights)} weights, {len(grads)} gradients and {len(momenta)} momenta")
    if scale not in _SCALES:
        raise ValueError(f"scale must be one of {_SCALES}, got {scale!r}")
    coef = _coefficients(coefficients, steps)
    lr, momentum, weight_decay = float(lr), float(momentum), float(weight_decay)
    if not (math.isfinite(lr) and lr >= 0 and 0 <= momentum < 1 and math.isfinite(weight_decay)
            and weight_decay >= 0):
        raise ValueError(f"lr {lr} and weight_decay {weight_decay} must be finite and not negative, "
                         f"momentum {momentum} in [0, 1)")
    if not weights:
        return
    first, rows, keep, back = weights[0], [], [], []
    dtype, index, scales = first.dtype, first.get_device(), {}
    for i, (w, g, m) in enumerate(zip(weights, grads, momenta)):
        shape = w.shape
        if w.dtype != dtype or dtype not in _DTYPES:
            raise TypeError(f"weights must share one of float16, bfloat16, float32; weight {i} is {w.dtype}")
        if len(shape) < 2:
            raise ValueError(f"weight {i} of shape {tuple(shape)} is not a matrix")
        if g.shape != shape or g.dtype != dtype:
            raise ValueError(f"gradient {i} must be {w.dtype} of shape {tuple(shape)}, got "
                             f"{g.dtype} {tuple(g.shape)}")
        if m.shape != shape or m.dtype != torch.float32:
            raise ValueError(f"momentum {i} must be float32 of shape {tuple(shape)}, got "
                             f"{m.dtype} {tuple(m.shape)}")
        n = w.numel()
        step = scales.get(shape)
        if step is None and n:
            _check_size(f"weight {i}", shape[0], n // shape[0])
            step = scales[shape] = lr * _scale(scale, shape[0], n // shape[0])
        if not (w.get_device() == g.get_device() == m.get_device() == index) or index < 0:
            backend.require_cuda(w, g, m)
            raise ValueError("weights, gradients and momenta must be on one device")
        if n == 0:
            continue
        wm, gm, mm = w, g, m
        if not (w.is_contiguous() and g.is_contiguous() and m.is_contiguous()):
            w_ = w.detach()
            wm = _rows_layout(w_)
            if wm is None:
                w_ = _copied(w, torch.empty(shape, dtype=dtype, device=w.device), f"weight {i}", back)
                wm = _rows_layout(w_)
            mm, gm = _like_layout(m.detach(), w_), _like_layout(g.detach(), w_)
            if mm is None:
                mm = _rows_layout(_copied(m, w_, f"momentum {i}", back))
            if gm is None:
                gm = _rows_layout(torch.empty_like(w_).copy_(g.detach()))
                keep.append(gm)
        r = shape[0]
        c = n // r
        rows.append((gm.data_ptr(), wm.data_ptr(), mm.data_ptr(), r, c, c, c, step))
    written = {p for row in rows for p in row[1:3]}
    written.update([t.data_ptr() for t, _ in back])
    if len(written) < 2 * len(rows) + len(back):
        raise ValueError("a weight or a momentum is given twice")
    # a gradient is read again after the momenta, and other weights, are written
    if not written.isdisjoint([row[0] for row in rows]) and any(
            row[0] in written and row[0] != row[1] for row in rows):
        raise ValueError("a gradient is also given as a momentum or as another weight")
    if not rows:
        return
    mats = b"".join([_MATRIX(*row) for row in rows])
    _run(backend.lib().fa_b200_muon_step, mats, len(rows), first, coef, steps, momentum,
         int(nesterov), 1.0 - lr * weight_decay)
    for t, c in back:
        t.copy_(c)
    # autograd notices weights that a graph still needs, as for torch's own updates
    torch.autograd.graph.increment_version(weights + momenta)


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for weight matrices (and convolution
    kernels, flattened to out x rest); see :func:`muon_step`.  Embeddings, norms
    and biases belong to another optimiser: parameters of fewer than two
    dimensions are refused."""

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95,
                 nesterov: bool = True, weight_decay: float = 0.0, scale: str = "aspect",
                 steps: int = 5, coefficients: Sequence = NEWTON_SCHULZ):
        if scale not in _SCALES:
            raise ValueError(f"scale must be one of {_SCALES}, got {scale!r}")
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError(f"bad lr {lr}, momentum {momentum} or weight_decay {weight_decay}")
        _coefficients(coefficients, steps)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, scale=scale, steps=steps,
                                      coefficients=coefficients))

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError(f"Muon updates matrices; got a parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # the base class casts state to its parameter's dtype; momentum stays float32
        # and takes its parameter's memory layout
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                buf = state_dict["state"].get(key, {}).get("momentum_buffer")
                if buf is None:
                    continue
                if buf.shape != p.shape:
                    raise ValueError(f"momentum of shape {tuple(buf.shape)} for a parameter of "
                                     f"shape {tuple(p.shape)}")
                self.state[p]["momentum_buffer"] = torch.empty_like(
                    p, dtype=torch.float32, requires_grad=False).copy_(buf.detach())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            sets: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                buf = state.get("momentum_buffer")
                if buf is None:
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
                elif buf.stride() != p.stride():  # the parameter was laid out anew
                    state["momentum_buffer"] = torch.empty_like(p, dtype=torch.float32).copy_(buf)
                ws, gs, ms = sets.setdefault((p.device, p.dtype), ([], [], []))
                ws.append(p)
                gs.append(p.grad)
                ms.append(state["momentum_buffer"])
            for ws, gs, ms in sets.values():
                muon_step(ws, gs, ms, **{k: group[k] for k in
                                         ("lr", "momentum", "nesterov", "weight_decay", "scale",
                                          "steps", "coefficients")})
        return loss
