"""Cases of a transformer block's operators with activations kept in 8 bits.

A network that restores whole frames keeps, for its backward pass, the inputs of
every norm, activation and product of every block: at 8160 tokens a 1920 x 1080
frame (16 x 16 patches) they fill the GPU long before its arithmetic is busy.
This file lists workloads of the operators that keep them in 8 bits (``listed``),
draws more of the same ranges (``draw``), and runs each either through the
package's entry points (``own`` true) or in a plain form of elementary float32
torch operations.

Kinds of case:

* ``norm``    ``fa.layer_norm``: residual sum and norm over the last dimension;
  with ``train`` its gradients, with ``keep8`` from an 8-bit copy of its input,
* ``pack``    ``fa.pack8`` and ``fa.unpack8``: an activation to 8 bits and back,
* ``gelu``    ``fa.gelu8``: the activation between the two products of an MLP, and
  its gradient from an 8-bit copy of its input,
* ``linear``  ``fa.linear8``: a product whose weight gradient reads an 8-bit copy
  of its input, forward and backward.

The 8-bit form: groups of 64 values of the last dimension hold their lowest value
``lo``, a power of two ``s`` and codes 0..255: ``s`` is the smallest (from 2^-126
up) with ``max - min <= 255 s`` and a value stands for ``code s + lo``.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
GROUP = 64
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #

def listed():
    return [
        # inference on a handful of tokens: latency is all there is
        {"name": "norm tokens f16", "kind": "norm", "dtype": "f16", "rows": 4, "width": 1024,
         "residual": True, "train": False, "keep8": False, "affine": "both"},
        # two 1920x1080 frames of 16x16 patches through a block's residual sum and norm
        {"name": "norm frames train bf16", "kind": "norm", "dtype": "bf16", "rows": 16320,
         "width": 1024, "residual": True, "train": True, "keep8": False, "affine": "both"},
        # odd token count and width in full precision, input kept in 8 bits
        {"name": "norm odd train f32 keep8", "kind": "norm", "dtype": "f32", "rows": 1551,
         "width": 577, "residual": False, "train": True, "keep8": True, "affine": "both"},
        # one frame through a wide network
        {"name": "norm wide train bf16 keep8", "kind": "norm", "dtype": "bf16", "rows": 8160,
         "width": 8192, "residual": True, "train": True, "keep8": True, "affine": "weight"},
        # the smallest activation: one row, a group and a part of one
        {"name": "pack row f32", "kind": "pack", "dtype": "f32", "rows": 1, "width": 200},
        # an MLP's hidden activation of eight frames
        {"name": "pack frames bf16", "kind": "pack", "dtype": "bf16", "rows": 65280,
         "width": 4096},
        # an MLP's activation on two frames
        {"name": "gelu frames train bf16", "kind": "gelu", "dtype": "bf16", "rows": 16320,
         "width": 4096, "approximate": "none"},
        # odd sizes in full precision, the tanh form
        {"name": "gelu odd train f32", "kind": "gelu", "dtype": "f32", "rows": 1551,
         "width": 1001, "approximate": "tanh"},
        # a small restoration network: eight 96x96 crops of 8x8 patches, width 192
        {"name": "linear crops train f32", "kind": "linear", "dtype": "f32", "rows": 1152,
         "inputs": 192, "outputs": 768, "bias": False},
        # odd sizes all round
        {"name": "linear odd train f16", "kind": "linear", "dtype": "f16", "rows": 1037,
         "inputs": 333, "outputs": 517, "bias": True},
        # the first product of an MLP on two frames
        {"name": "linear up train bf16", "kind": "linear", "dtype": "bf16", "rows": 16320,
         "inputs": 1024, "outputs": 4096, "bias": True},
        # the second, on four frames
        {"name": "linear down train bf16", "kind": "linear", "dtype": "bf16", "rows": 32640,
         "inputs": 4096, "outputs": 1024, "bias": True},
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "pack", "gelu", "linear", "linear"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "linear":
        # no more than the largest listed product; float32 an eighth of it
        most = 1.3e11 if dtype != "f32" else 1.6e10
        inputs, outputs = _size(rng, 16, 5000), _size(rng, 16, 5000)
        if rng.random() < 0.5:  # widths are mostly whole vectors
            inputs, outputs = (inputs + 7) // 8 * 8, (outputs + 7) // 8 * 8
        rows = _size(rng, 1, min(60000, most / (inputs * outputs)))
        return {"kind": kind, "dtype": dtype, "rows": rows, "inputs": inputs,
                "outputs": outputs, "bias": rng.random() < 0.6}
    width = _size(rng, 24, 12000)
    if rng.random() < 0.6:
        width = (width + 7) // 8 * 8
    rows = _size(rng, 1, min(70000, 6.5e7 / width))
    if kind == "norm":
        train = rng.random() < 0.75
        return {"kind": kind, "dtype": dtype, "rows": rows, "width": width,
                "residual": rng.random() < 0.5, "train": train,
                "keep8": train and rng.random() < 0.5,
                "affine": rng.choice(("both", "both", "weight", "none"))}
    if kind == "gelu":
        return {"kind": kind, "dtype": dtype, "rows": rows, "width": width,
                "approximate": rng.choice(("none", "none", "tanh"))}
    return {"kind": kind, "dtype": dtype, "rows": rows, "width": width}


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #

def _stream(rows, width, g):
    """Activations: channels of different strength and offset, a few far above the rest."""
    strength = torch.exp(0.5 * torch.randn(width, generator=g, device="cuda"))
    strength = strength * (1 + 9 * (torch.rand(width, generator=g, device="cuda") < 0.01).float())
    offset = 0.3 * torch.randn(width, generator=g, device="cuda")
    return torch.randn(rows, width, generator=g, device="cuda") * strength + offset


def _grad(rows, width, g):
    return 1e-2 * torch.randn(rows, width, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "linear":
        t, k, m = case["rows"], case["inputs"], case["outputs"]
        s["x"] = _stream(t, k, g).to(dtype)
        s["weight"] = (torch.randn(m, k, generator=g, device="cuda") / math.sqrt(k)).to(dtype)
        s["bias"] = None
        if case["bias"]:
            s["bias"] = (0.1 * torch.randn(m, generator=g, device="cuda")).to(dtype)
        s["grad"] = _grad(t, m, g).to(dtype)
        leaves = ("x", "weight", "bias")
    elif case["kind"] == "norm":
        t, n = case["rows"], case["width"]
        s["x"] = _stream(t, n, g).to(dtype)
        s["residual"] = _stream(t, n, g).to(dtype) if case["residual"] else None
        s["weight"] = s["bias"] = None
        if case["affine"] != "none":
            s["weight"] = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(dtype)
        if case["affine"] == "both":
            s["bias"] = (0.2 * torch.randn(n, generator=g, device="cuda")).to(dtype)
        if case["train"]:
            s["grad"] = _grad(t, n, g).to(dtype)
            if case["residual"]:
                s["grad_sum"] = _grad(t, n, g).to(dtype)
        leaves = ("x", "residual", "weight", "bias") if case["train"] else ()
    else:
        s["x"] = _stream(case["rows"], case["width"], g).to(dtype)
        if case["kind"] == "gelu":
            s["grad"] = _grad(case["rows"], case["width"], g).to(dtype)
        leaves = ("x",) if case["kind"] == "gelu" else ()
    for name in leaves:
        if s[name] is not None:
            s[name].requires_grad_(True)
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #

def run(state):
    case = state["case"]
    return {"norm": _run_norm, "pack": _run_pack, "gelu": _run_gelu,
            "linear": _run_linear}[case["kind"]](case, state)


def _kept(x):
    """What the 8-bit copy of x stands for, float32: x in groups along its rows."""
    rows, width = x.shape
    groups = (width + GROUP - 1) // GROUP
    short = groups * GROUP - width
    if short:  # the last value again: it changes no group's range
        x = torch.cat((x, x[:, -1:].expand(rows, short)), 1)
    v = x.float().view(rows, groups, GROUP)
    lo = v.amin(-1, keepdim=True)
    d = v.amax(-1, keepdim=True) - lo
    part, power = torch.frexp(d)  # d = part 2^power, part in [1/2, 1)
    power = torch.where(part <= 255 / 256, power - 8, power - 7).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(d), power)
    v = torch.round((v - lo) / s) * s + lo
    return v.view(rows, groups * GROUP)[:, :width].to(x.dtype).float()


def _run_norm(case, s):
    if own:
        import frame_analytics_b200 as fa
        got = fa.layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS,
                            keep8=case["keep8"])
        out = dict(zip(("y", "sum"), got if case["residual"] else (got,)))
        if not case["train"]:
            return out
        names = [n for n in ("x", "residual", "weight", "bias") if s[n] is not None]
        grads = torch.autograd.grad(tuple(out.values()), [s[n] for n in names],
                                    [s["grad"]] + ([s["grad_sum"]] if case["residual"] else []))
        return {**{k: v.detach() for k, v in out.items()},
                **{"grad_" + n: g for n, g in zip(names, grads)}}
    x, out = s["x"].detach(), {}
    dtype = x.dtype
    if case["residual"]:
        x = (x.float() + s["residual"].detach().float()).to(dtype)
        out["sum"] = x
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    r = torch.rsqrt((xf - mean).square().mean(-1, keepdim=True) + EPS)
    w = 1.0 if s["weight"] is None else s["weight"].detach().float()
    y = (xf - mean) * r * w
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    out = {"y": y.to(dtype), **out}
    if case["train"]:
        xh = ((_kept(x) if case["keep8"] else xf) - mean) * r
        dy = s["grad"].float()
        g = dy * w
        dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        if case["residual"]:
            dx = dx + s["grad_sum"].float()
        out["grad_x"] = dx.to(dtype)
        if case["residual"]:
            out["grad_residual"] = out["grad_x"]
        if s["weight"] is not None:
            out["grad_weight"] = (dy * xh).sum(0).to(dtype)
        if s["bias"] is not None:
            out["grad_bias"] = dy.sum(0).to(dtype)
    return out


def _run_pack(case, s):
    if own:
        import frame_analytics_b200 as fa
        return fa.unpack8(fa.pack8(s["x"]))
    return _kept(s["x"]).to(s["x"].dtype)


def _gelu(x, approximate):
    """Value and derivative, float32."""
    if approximate == "tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return (0.5 * x * (1 + t),
                0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x))
    p = 0.5 * torch.erfc(x * -math.sqrt(0.5))
    return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def _run_gelu(case, s):
    if own:
        import frame_analytics_b200 as fa
        y = fa.gelu8(s["x"], approximate=case["approximate"])
        return {"y": y.detach(), "grad_x": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    x = s["x"].detach()
    return {"y": _gelu(x.float(), case["approximate"])[0].to(x.dtype),
            "grad_x": (s["grad"].float() * _gelu(_kept(x), case["approximate"])[1]).to(x.dtype)}


def _run_linear(case, s):
    if own:
        import frame_analytics_b200 as fa
        y = fa.linear8(s["x"], s["weight"], s["bias"])
        names = [n for n in ("x", "weight", "bias") if s[n] is not None]
        grads = torch.autograd.grad(y, [s[n] for n in names], s["grad"])
        return {"y": y.detach(), **{"grad_" + n: g for n, g in zip(names, grads)}}
    x, w, dy = s["x"].detach(), s["weight"].detach(), s["grad"].float()
    y = torch.matmul(x.float(), w.float().mT)
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    out = {"y": y.to(x.dtype), "grad_x": torch.matmul(dy, w.float()).to(x.dtype),
           "grad_weight": torch.matmul(dy.mT, _kept(x)).to(x.dtype)}
    if s["bias"] is not None:
        out["grad_bias"] = dy.sum(0).to(x.dtype)
    return out


# --------------------------------------------------------------------------- #
# what a pass cannot do without, and its values in 64 bits
# --------------------------------------------------------------------------- #

def work(case):
    e = DTYPES[case["dtype"]].itemsize
    # codes, and the lowest value and the power of each group
    kept = 1 + (4 if e == 2 else 8) / GROUP
    if case["kind"] == "linear":
        t, k, m = case["rows"], case["inputs"], case["outputs"]
        # forward: x, W, y, the kept copy; backward: dy, W, the copy, dx, dW
        size = e * (2 * t * k + 3 * m * k + 2 * t * m) + 2 * t * k * kept
        if case["bias"]:
            size += 2 * e * m
        return {"bytes": size, "flops": 6.0 * t * k * m}
    n = case["rows"] * case["width"]
    if case["kind"] == "pack":
        return {"bytes": n * (2 * e + 2 * kept), "flops": 8 * n}
    if case["kind"] == "gelu":
        return {"bytes": n * (4 * e + 2 * kept), "flops": 40 * n}
    parts = 4 if case["residual"] else 2
    size, flops = parts * n * e, 8 * n
    if case["train"]:  # dy (and the sum's gradient) in, dx out, what was kept
        size += (parts // 2 + 1) * n * e + (2 * n * kept if case["keep8"] else n * e)
        flops += 14 * n
    return {"bytes": size, "flops": flops}


def _exact_kept(x):
    """The 8-bit copy's values in float64, group by group position: x (rows, width)
    in its own type."""
    wide, kept = x.double(), torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[1], GROUP):
        v = wide[:, first:first + GROUP]
        lo, hi = v.min(1, keepdim=True).values, v.max(1, keepdim=True).values
        d = (hi - lo).float().double()  # differences are rounded to float32
        e = torch.ceil(torch.log2((d / 255).clamp(min=2.0 ** -126)))
        # the logarithm may be one off at a power of two
        e = torch.where(d <= 255 * torch.exp2(e - 1), e - 1, e)
        e = torch.where(d > 255 * torch.exp2(e), e + 1, e).clamp(min=-126)
        s = torch.exp2(e)
        kept[:, first:first + GROUP] = ((v - lo).float().double() / s).round() * s + lo
    return kept.to(x.dtype).double()


def _exact_gelu(x, approximate):
    if approximate == "tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x ** 3)))
    return x * torch.special.ndtr(x)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    if case["kind"] == "pack":
        return _exact_kept(x)
    dy = s["grad"].double() if "grad" in s else None
    if case["kind"] == "gelu":
        at = _exact_kept(x).requires_grad_(True)
        grad, = torch.autograd.grad(_exact_gelu(at, case["approximate"]), at, dy)
        return {"y": _exact_gelu(x.double(), case["approximate"]), "grad_x": grad}
    w = None if s["weight"] is None else s["weight"].detach().double()
    b = None if s["bias"] is None else s["bias"].detach().double()
    if case["kind"] == "linear":
        out = {"y": x.double() @ w.T, "grad_x": dy @ w, "grad_weight": dy.T @ _exact_kept(x)}
        if b is not None:
            out["y"] += b
            out["grad_bias"] = dy.sum(0)
        return out
    out = {}
    if case["residual"]:
        x = (x.double() + s["residual"].detach().double()).to(x.dtype)
    wide = x.double()
    var, mean = torch.var_mean(wide, dim=1, correction=0, keepdim=True)
    scale = (var + EPS).sqrt()
    xh = (wide - mean) / scale
    y = xh if w is None else xh * w
    out["y"] = y if b is None else y + b
    if case["residual"]:
        out["sum"] = wide
    if case["train"]:
        if case["keep8"]:
            xh = (_exact_kept(x) - mean) / scale
        g = dy if w is None else dy * w
        width = case["width"]
        dx = (g - g.sum(1, keepdim=True) / width
              - xh * torch.linalg.vecdot(g, xh).unsqueeze(1) / width) / scale
        if case["residual"]:
            dx = dx + s["grad_sum"].double()
            out["grad_x"] = out["grad_residual"] = dx
        else:
            out["grad_x"] = dx
        if w is not None:
            out["grad_weight"] = torch.einsum("tn,tn->n", dy, xh)
        if b is not None:
            out["grad_bias"] = torch.einsum("tn->n", dy)
    return out
