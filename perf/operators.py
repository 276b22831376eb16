"""Cases of the training-step operators: orthogonalised updates and attention operands.

A model that is trained against the package's losses needs two more things
around them on the GPU: the queries and keys of its attention layers, normalised
and rotated by position, and the optimiser's update of its weight matrices.  This
file lists workloads of those operators (``listed``), draws more of the same
ranges (``draw``), and runs each either through the package's entry points
(``own`` true) or in a plain form of elementary float32 torch operations.

Kinds of case:

* ``orth``  ``fa.orthogonalize``: Newton-Schulz orthogonalisation of a stack of
  matrices,
* ``muon``  ``fa.muon_step``: momentum, orthogonalisation and weight update of a
  list of matrices in place,
* ``qk``    ``fa.qk_norm_rotary``: norm of each query and key head and rotation
  by position; with ``train`` also its gradients.
"""

from __future__ import annotations

import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MOMENTUM, DECAY, EPS = 0.02, 0.95, 0.01, 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #

def listed():
    return [
        # one small layer's gradient: launch latency is all there is
        {"name": "orth 64x64 bf16", "kind": "orth", "dtype": "bf16", "batch": 1, "rows": 64,
         "cols": 64},
        # odd sizes in full precision, a stack of three
        {"name": "orth 3x 201x333 f32", "kind": "orth", "dtype": "f32", "batch": 3, "rows": 201,
         "cols": 333},
        # one kind of projection of every layer of a mid-size model, stacked
        {"name": "orth 12x 768x768 bf16", "kind": "orth", "dtype": "bf16", "batch": 12,
         "rows": 768, "cols": 768},
        # a packed projection, taller than wide, full precision
        {"name": "orth 2304x768 f32", "kind": "orth", "dtype": "f32", "batch": 1, "rows": 2304,
         "cols": 768},
        # the largest matrix of a large model
        {"name": "orth 4096x8192 bf16", "kind": "orth", "dtype": "bf16", "batch": 1,
         "rows": 4096, "cols": 8192},
        # every matrix of a small restoration network: convolution kernels (flattened to
        # out x in*kh*kw), square projections and both halves of its MLPs; float32 weights
        {"name": "muon small net f32", "kind": "muon", "dtype": "f32",
         "shapes": "6*64x576,4*180x180,2*360x180,2*180x360"},
        # layers of a large one, weights in bfloat16 with float32 momentum
        {"name": "muon large net bf16", "kind": "muon", "dtype": "bf16",
         "shapes": "4*2048x2048,1*5632x2048,1*2048x5632"},
        # one new token of a few sequences (serving): latency
        {"name": "qk token bf16", "kind": "qk", "train": False, "dtype": "bf16", "batch": 4,
         "length": 1, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "table": 4096, "weights": "dim"},
        # a long prompt, forward alone, grouped key heads
        {"name": "qk long f16", "kind": "qk", "train": False, "dtype": "f16", "batch": 1,
         "length": 32761, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "table": 40000, "weights": "dim"},
        # training on 1920x1080 frames cut into 16x16 patches (120 x 68 tokens)
        {"name": "qk frames train bf16", "kind": "qk", "train": True, "dtype": "bf16",
         "batch": 2, "length": 8160, "q_heads": 16, "k_heads": 16, "dim": 64, "rotary": 64,
         "interleaved": False, "table": 8160, "weights": "dim"},
        # training in full precision: odd length, part of the head rotated in adjacent
        # pairs, a weight for each head
        {"name": "qk odd train f32", "kind": "qk", "train": True, "dtype": "f32", "batch": 3,
         "length": 517, "q_heads": 6, "k_heads": 2, "dim": 96, "rotary": 48,
         "interleaved": True, "table": 1024, "weights": "head"},
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v + 1 if v == 3 << 10 else v


def draw(rng):
    kind = rng.choice(("orth", "orth", "muon", "qk", "qk"))
    if kind == "orth":
        rows, cols = _size(rng, 16, 5000), _size(rng, 16, 5000)
        small, large = min(rows, cols), max(rows, cols)
        most = max(1, min(24, int(2.0e11 / (3 * small * small * large + small ** 3))))
        return {"kind": "orth", "dtype": rng.choice(("bf16", "bf16", "f32", "f16")),
                "batch": _size(rng, 1, most), "rows": rows, "cols": cols}
    if kind == "muon":
        groups = []
        for _ in range(rng.randint(1, 4)):
            groups.append("%d*%dx%d" % (rng.randint(1, 6), _size(rng, 32, 1500),
                                        _size(rng, 32, 1500)))
        return {"kind": "muon", "dtype": rng.choice(("bf16", "f32")),
                "shapes": ",".join(groups)}
    dim = rng.choice((32, 48, 64, 80, 96, 128, 192, 256))
    k_heads = rng.choice((1, 2, 4, 8))
    q_heads = k_heads * rng.choice((1, 2, 3, 4))
    batch = _size(rng, 1, 16)
    length = _size(rng, 1, max(2, int(1.2e8 / (batch * (q_heads + k_heads) * dim))))
    length = min(length, 60000)
    return {"kind": "qk", "train": rng.random() < 0.5,
            "dtype": rng.choice(("bf16", "f16", "f32")), "batch": batch, "length": length,
            "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "rotary": dim if rng.random() < 0.7 else dim // 2,
            "interleaved": rng.random() < 0.4, "table": length + rng.randint(0, 1000),
            "weights": rng.choice(("dim", "head", "none"))}


def _shapes(case):
    out = []
    for group in case["shapes"].split(","):
        count, shape = group.split("*")
        rows, cols = shape.split("x")
        out += [(int(rows), int(cols))] * int(count)
    return out


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #

def _gradient(batch, rows, cols, g):
    """A stack of gradient-like matrices: a few strong directions whose strength
    falls off, over a floor of noise."""
    rank = max(1, min(32, rows // 4, cols // 4))
    u = torch.randn(batch, rows, rank, generator=g, device="cuda")
    v = torch.randn(batch, rank, cols, generator=g, device="cuda")
    fall = torch.arange(1, rank + 1, device="cuda", dtype=torch.float32) ** -1.0
    noise = torch.randn(batch, rows, cols, generator=g, device="cuda")
    return 1e-3 * (torch.matmul(u * fall, v) + noise)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "orth":
        x = _gradient(case["batch"], case["rows"], case["cols"], g).to(dtype)
        return {"case": case, "x": x[0] if case["batch"] == 1 else x}
    if case["kind"] == "muon":
        w, d, m = [], [], []
        for rows, cols in _shapes(case):
            w.append((torch.randn(rows, cols, generator=g, device="cuda")
                      / math.sqrt(cols)).to(dtype))
            d.append(_gradient(1, rows, cols, g)[0].to(dtype))
            m.append(5 * _gradient(1, rows, cols, g)[0])
        return {"case": case, "weights": w, "grads": d, "momenta": m}
    b, n, hq, hk, dim = (case[k] for k in ("batch", "length", "q_heads", "k_heads", "dim"))
    # queries, keys and values come packed out of one projection
    packed = torch.randn(b, n, hq + 2 * hk, dim, generator=g, device="cuda").to(dtype)
    half = case["rotary"] // 2
    angle = (torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None]
             * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
    first = torch.randint(0, case["table"] - n + 1, (b, 1), generator=g, device="cuda")
    s = {"case": case, "q": packed[:, :, :hq], "k": packed[:, :, hq:hq + hk],
         "cos": angle.cos().float(), "sin": angle.sin().float(),
         "positions": first + torch.arange(n, device="cuda"), "q_weight": None,
         "k_weight": None}
    if case["weights"] != "none":
        per_head = case["weights"] == "head"
        for name, heads in (("q_weight", hq), ("k_weight", hk)):
            shape = (heads, dim) if per_head else (dim,)
            s[name] = (1 + 0.2 * torch.randn(shape, generator=g, device="cuda")).to(dtype)
    if case["train"]:
        s["grad_q"] = (1e-2 * torch.randn(b, n, hq, dim, generator=g, device="cuda")).to(dtype)
        s["grad_k"] = (1e-2 * torch.randn(b, n, hk, dim, generator=g, device="cuda")).to(dtype)
        for name in ("q", "k", "q_weight", "k_weight"):
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_(True)
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #

def run(state):
    case = state["case"]
    return {"orth": _run_orth, "muon": _run_muon, "qk": _run_qk}[case["kind"]](case, state)


def _newton_schulz(x):
    """Float32 [..., m, n]: odd polynomial steps on x over its Frobenius norm."""
    a, b, c = COEFFICIENTS
    norm = x.square().sum(dim=(-2, -1), keepdim=True).sqrt()
    x = torch.where(norm > 0, x / norm, torch.zeros_like(x))
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-2, -1) if tall else x


def _run_orth(case, s):
    if own:
        import frame_analytics_b200 as fa
        return fa.orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS)
    return _newton_schulz(s["x"].float()).to(s["x"].dtype)


def _run_muon(case, s):
    if own:
        import frame_analytics_b200 as fa
        fa.muon_step(s["weights"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM,
                     nesterov=True, weight_decay=DECAY, scale="aspect", steps=STEPS,
                     coefficients=COEFFICIENTS)
    else:
        for w, g, m in zip(s["weights"], s["grads"], s["momenta"]):
            g = g.float()
            m.mul_(MOMENTUM).add_(g)
            o = _newton_schulz(g + MOMENTUM * m)
            rows, cols = w.shape
            w.copy_(w.float() * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, rows / cols)) * o)
    return {"weights": s["weights"], "momenta": s["momenta"]}


def _rotate(x, cos, sin, interleaved):
    """Float32 [b, n, h, d]; cos, sin [b, n, 1, r/2].  Rotates the first r components."""
    half = cos.shape[-1]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        x1, x2 = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1).flatten(-2)
    else:
        x1, x2 = head[..., :half], head[..., half:]
        turned = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)
    return torch.cat((turned, rest), -1)


def _run_qk(case, s):
    if own:
        import frame_analytics_b200 as fa
        q, k = fa.qk_norm_rotary(s["q"], s["k"], s["cos"], s["sin"], q_weight=s["q_weight"],
                                 k_weight=s["k_weight"], eps=EPS, positions=s["positions"],
                                 interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": q, "k": k}
        names = [n for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None]
        grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["grad_q"], s["grad_k"]))
        return {"q": q.detach(), "k": k.detach(),
                **{"grad_" + n: g for n, g in zip(names, grads)}}
    out = {}
    cos = s["cos"][s["positions"]][:, :, None]
    sin = s["sin"][s["positions"]][:, :, None]
    for name in ("q", "k"):
        x, w = s[name].detach(), s[name + "_weight"]
        w = None if w is None else w.detach()
        xf = x.float()
        r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
        xhat = xf * r
        wf = 1.0 if w is None else w.float()
        out[name] = _rotate(xhat * wf, cos, sin, case["interleaved"]).to(x.dtype)
        if case["train"]:
            g = _rotate(s["grad_" + name].float(), cos, -sin, case["interleaved"])
            gx = g * wf
            gx = r * (gx - xhat * (gx * xhat).mean(-1, keepdim=True))
            out["grad_" + name] = gx.to(x.dtype)
            if w is not None:
                gw = (g * xhat).sum(dim=(0, 1) if w.dim() == 2 else (0, 1, 2))
                out["grad_" + name + "_weight"] = gw.to(w.dtype)
    return out


# --------------------------------------------------------------------------- #
# what a pass cannot do without, and its values in 64 bits
# --------------------------------------------------------------------------- #

def _orth_flops(rows, cols):
    # the Gram matrix and its square are symmetric: half of each product
    small, large = min(rows, cols), max(rows, cols)
    return STEPS * (3.0 * small * small * large + float(small) ** 3)


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "orth":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * n * e, "flops": case["batch"] * _orth_flops(case["rows"],
                                                                         case["cols"])}
    if case["kind"] == "muon":
        n = sum(r * c for r, c in _shapes(case))
        return {"bytes": n * (3 * e + 8),
                "flops": sum(_orth_flops(r, c) for r, c in _shapes(case))}
    heads = case["q_heads"] + case["k_heads"]
    tokens = case["batch"] * case["length"]
    n = tokens * heads * case["dim"]
    tables = min(tokens, case["table"]) * case["rotary"] * 4 + tokens * 8
    if case["train"]:  # forward reads and writes; backward reads x and dy, writes dx
        return {"bytes": 5 * n * e + 2 * tables, "flops": 25 * n}
    return {"bytes": 2 * n * e + tables, "flops": 9 * n}


def _exact_orth(x):
    """The composed polynomial on the Gram matrix's eigenvalues, times x."""
    a, b, c = COEFFICIENTS
    if not bool(x.any()):
        return x
    x = x / torch.linalg.matrix_norm(x)
    tall = x.shape[0] > x.shape[1]
    lam, v = torch.linalg.eigh(x.mT @ x if tall else x @ x.mT)
    factor = torch.ones_like(lam)
    for _ in range(STEPS):
        p = a + lam * (b + c * lam)
        factor, lam = factor * p, lam * p * p
    return (x @ v) * factor @ v.mT if tall else v @ (factor[:, None] * (v.mT @ x))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "orth":
        x = s["x"].double()
        if x.dim() == 2:
            return _exact_orth(x)
        return torch.stack([_exact_orth(m) for m in x])
    if case["kind"] == "muon":
        weights, momenta = [], []
        for w, g, m in zip(s["weights"], s["grads"], s["momenta"]):
            w, g, m = w.double(), g.double(), m.double()
            momenta.append(g + MOMENTUM * m)
            o = _exact_orth(g + MOMENTUM * momenta[-1])
            weights.append(w - LR * (DECAY * w + max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * o))
        return {"weights": weights, "momenta": momenta}
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, :, None]
    half = case["rotary"] // 2
    out = {}
    for name in ("q", "k"):
        x = s[name].detach().double().requires_grad_(case["train"])
        w = s[name + "_weight"]
        w = None if w is None else w.detach().double().requires_grad_(case["train"])
        y = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).pow(0.5)
        y = y if w is None else y * w
        if case["interleaved"]:
            z = torch.complex(y[..., 0:2 * half:2], y[..., 1:2 * half:2]) * turn
            turned = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
            turned = torch.cat((z.real, z.imag), -1)
        y = torch.cat((turned, y[..., 2 * half:]), -1)
        out[name] = y.detach()
        if case["train"]:
            leaves = [x] if w is None else [x, w]
            grads = torch.autograd.grad(y, leaves, s["grad_" + name].double())
            out["grad_" + name] = grads[0]
            if w is not None:
                out["grad_" + name + "_weight"] = grads[1]
        del x, y, z, turned
    return out
