"""The training-step operators on the GPU, against plain float64 formulas.

Tolerances: u is the unit roundoff of the output's type (2^-24, 2^-11, 2^-8
for float32, float16, bfloat16).  Each output is rounded once (u relative per
value); the sums behind it are float32 over n terms, whose error stays below
n 2^-24 of the sum of magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

import frame_analytics_b200 as fa
from frame_analytics_b200.optim import NEWTON_SCHULZ

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# --------------------------------------------------------------------------- #
# query / key norm and rotation
# --------------------------------------------------------------------------- #

def tables(positions, rotary, device="cuda"):
    half = rotary // 2
    a = (torch.arange(positions, dtype=torch.float64, device=device)[:, None]
         * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half))
    return a.cos().float(), a.sin().float()


def plain_qk(x, cos, sin, w, eps, positions, interleaved):
    """float64, differentiable."""
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w
    if cos is None:
        return y
    if positions is None:
        positions = torch.arange(x.shape[1], device=x.device)
    c, s = (t.double()[positions.long()] for t in (cos, sin))
    if c.dim() == 2:
        c, s = c[None], s[None]
    c, s = c[:, :, None], s[:, :, None]
    r = 2 * cos.shape[1]
    i1 = slice(0, r, 2) if interleaved else slice(0, r // 2)
    i2 = slice(1, r, 2) if interleaved else slice(r // 2, r)
    out = y.clone()
    out[..., i1] = y[..., i1] * c - y[..., i2] * s
    out[..., i2] = y[..., i2] * c + y[..., i1] * s
    return out


def close(got, want, u, terms):
    """|got - want| within one rounding plus float32 sums of `terms` terms, on the
    scale of the output (its largest value: sums may cancel)."""
    want = want.double()
    err = (got.double() - want).abs()
    tol = u * want.abs() + (8 + terms) * 2.0 ** -24 * want.abs().max().clamp_min(1e-30)
    if u == 2.0 ** -11:
        tol = tol + 2.0 ** -25  # float16's subnormal spacing
    assert bool((err <= tol).all()), (err / tol).max().item()


# batch, length, q heads, k heads, dim, rotary, interleaved, weights
QK = [
    (1, 1, 1, 1, 64, 64, False, "dim"),
    (4, 1, 8, 2, 128, 128, False, "dim"),
    (2, 33, 4, 4, 64, 64, True, "dim"),
    (3, 17, 3, 1, 80, 80, False, "head"),
    (2, 9, 4, 2, 96, 48, True, "head"),
    (2, 40, 5, 5, 48, 24, False, "none"),
    (1, 301, 2, 1, 256, 256, False, "dim"),
    (2, 5, 2, 3, 7, 6, False, "dim"),      # odd head size: two components pass or turn alone
    (1, 6, 1, 2, 1, 0, False, "dim"),
    (2, 3, 2, 2, 33, 20, True, "head"),
    (1, 4, 2, 1, 512, 512, False, "dim"),
    (1, 4, 2, 1, 130, 130, True, "dim"),
    (2, 65, 6, 2, 128, 0, False, "dim"),
    (70, 2, 2, 2, 32, 32, False, "head"),
]


def qk_case(case, dtype, seed=0, w_dtype=None):
    b, n, hq, hk, d, r, inter, weights = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    packed = torch.randn(b, n, hq + 2 * hk, d, generator=g, device="cuda").to(dtype)
    q, k = packed[:, :, :hq], packed[:, :, hq:hq + hk]
    cos, sin = tables(n + 11, r) if r else (None, None)
    pos = torch.randint(0, n + 11, (b, n), generator=g, device="cuda") if r else None
    ws = [None, None]
    if weights != "none":
        ws = [(1 + 0.3 * torch.randn((h, d) if weights == "head" else (d,), generator=g,
                                     device="cuda")).to(w_dtype or dtype) for h in (hq, hk)]
    gs = [torch.randn(b, n, h, d, generator=g, device="cuda").to(dtype) for h in (hq, hk)]
    return q, k, cos, sin, pos, ws, gs, inter


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", QK)
def test_qk_forward(case, dtype):
    q, k, cos, sin, pos, (qw, kw), _, inter = qk_case(case, dtype)
    got = fa.qk_norm_rotary(q, k, cos, sin, q_weight=qw, k_weight=kw, positions=pos,
                            interleaved=inter, eps=1e-5)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        want = plain_qk(x.double(), cos, sin, None if w is None else w.double(), 1e-5, pos, inter)
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        close(y, want, U[dtype], 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", QK)
def test_qk_backward(case, dtype):
    q, k, cos, sin, pos, ws, gs, inter = qk_case(case, dtype, seed=1)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, *ws) if t is not None]
    qw, kw = leaves[2:] if len(leaves) == 4 else (None, None)
    out = fa.qk_norm_rotary(leaves[0], leaves[1], cos, sin, q_weight=qw, k_weight=kw,
                            positions=pos, interleaved=inter, eps=1e-5)
    got = torch.autograd.grad(out, leaves, gs)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    wqw, wkw = wide[2:] if len(wide) == 4 else (None, None)
    ref = (plain_qk(wide[0], cos, sin, wqw, 1e-5, pos, inter),
           plain_qk(wide[1], cos, sin, wkw, 1e-5, pos, inter))
    want = torch.autograd.grad(ref, wide, [g.double() for g in gs])
    tokens = q.shape[0] * q.shape[1]
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.shape == b.shape and a.dtype == leaves[i].dtype
        if i < 2:
            close(a, b, U[dtype], 16)
        else:  # sums over tokens (and heads) of terms of order 1, with either sign
            n = tokens * (1 if b.dim() == 2 else (q, k)[i - 2].shape[2])
            err = (a.double() - b).abs()
            tol = U[dtype] * b.abs() + 2.0 ** -24 * (8 + n) * 4 * math.sqrt(n)
            assert bool((err <= tol).all()), (err / tol).max().item()


def test_qk_gradient_against_differences():
    """Central differences of the float64 plain form's scalar, with the kernel's
    own float32 gradient: the difference quotient is good to h^2."""
    q, k, cos, sin, pos, ws, gs, inter = qk_case((1, 3, 2, 1, 16, 8, True, "head"),
                                                 torch.float32, seed=5)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *ws)]
    out = fa.qk_norm_rotary(leaves[0], leaves[1], cos, sin, q_weight=leaves[2],
                            k_weight=leaves[3], positions=pos, interleaved=inter)
    grads = torch.autograd.grad(out, leaves, gs)

    def value(ts):
        t = [u.double() for u in ts]
        return float((plain_qk(t[0], cos, sin, t[2], 1e-6, pos, inter) * gs[0]).sum()
                     + (plain_qk(t[1], cos, sin, t[3], 1e-6, pos, inter) * gs[1]).sum())

    h = 1e-4
    for i, leaf in enumerate(leaves):
        flat = leaf.detach().double().flatten()
        for j in range(0, flat.numel(), 5):
            vals = []
            for sgn in (1, -1):
                moved = flat.clone()
                moved[j] += sgn * h
                ts = [t.detach().double() for t in leaves]
                ts[i] = moved.view(leaf.shape)
                vals.append(value(ts))
            fd = (vals[0] - vals[1]) / (2 * h)
            assert abs(fd - float(grads[i].flatten()[j])) < 2e-5 * (1 + abs(fd))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_qk_float32_weights_and_their_gradient(dtype):
    q, k, cos, sin, pos, ws, gs, inter = qk_case(QK[2], dtype, w_dtype=torch.float32)
    ws = [w.requires_grad_(True) for w in ws]
    out = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos,
                            interleaved=inter)
    got = torch.autograd.grad(out, ws, gs)
    wide = [w.detach().double().requires_grad_(True) for w in ws]
    ref = [plain_qk(x.double(), cos, sin, w, 1e-6, pos, inter) for x, w in zip((q, k), wide)]
    want = torch.autograd.grad(ref, wide, [g.double() for g in gs])
    for a, b in zip(got, want):
        assert a.dtype == torch.float32
        assert float((a.double() - b).abs().max()) < 2.0 ** -24 * 400 * float(b.abs().max())


def test_qk_default_positions_int32_and_broadcast_agree():
    q, k, cos, sin, _, ws, _, _ = qk_case(QK[2], torch.bfloat16)
    n = q.shape[1]
    a = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1])
    row = torch.arange(n, device="cuda")
    for p in (row, row.int(), row.expand(2, n), row.repeat(2, 1).int()):
        b = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=p)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dim,rotary", [(64, 64), (33, 20)])
def test_qk_positions_outside_the_tables_give_nan_rows(dim, rotary):
    q, k, cos, sin, _, ws, gs, _ = qk_case((2, 4, 2, 1, dim, rotary, False, "dim"), torch.float32)
    P = cos.shape[0]
    pos = torch.tensor([[0, P, 1, -1], [P - 1, 2, 1 << 40, -(1 << 40)]], device="cuda")
    bad = (pos < 0) | (pos >= P)
    qg = q.detach().requires_grad_(True)
    y = fa.qk_norm_rotary(qg, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    (dq,) = torch.autograd.grad(y[0], qg, gs[0])
    for t in (*y, dq):
        assert bool(t[bad].isnan().all()) and bool(t[~bad].isfinite().all())


def test_qk_out_in_place_strided_and_cache_slice():
    q, k, cos, sin, pos, ws, _, _ = qk_case((3, 1, 4, 2, 64, 64, False, "dim"), torch.bfloat16)
    want = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    cache = torch.zeros(3, 2, 50, 64, dtype=torch.bfloat16, device="cuda")  # (B, Hk, L, D)
    slot = cache[:, :, 7:8].transpose(1, 2)
    q_in = q.clone()
    got = fa.qk_norm_rotary(q_in, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos,
                            out=(q_in, slot))
    assert got[0] is q_in and torch.equal(q_in, want[0])
    assert torch.equal(cache[:, :, 7], want[1][:, 0]) and int(cache.count_nonzero()) == \
        int(want[1].count_nonzero())
    for dim, rot in ((512, 512), (33, 20)):
        q, k, cos, sin, pos, ws, _, _ = qk_case((2, 3, 2, 1, dim, rot, False, "dim"), torch.float32)
        want = fa.qk_norm_rotary(q, k, cos, sin, positions=pos)
        q, k = q.clone(), k.clone()
        fa.qk_norm_rotary(q, k, cos, sin, positions=pos, out=(q, k))
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_qk_misaligned_and_non_unit_stride_inputs_agree():
    q, k, cos, sin, pos, ws, _, _ = qk_case((2, 6, 2, 2, 64, 64, False, "dim"), torch.bfloat16)
    want = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    store = torch.empty(2 * 6 * 2 * 65 + 1, dtype=torch.bfloat16, device="cuda")
    odd = store[1:].view(2, 6, 2, 65)[..., :64].copy_(q)
    swapped = k.transpose(1, 3).contiguous().transpose(1, 3)
    got = fa.qk_norm_rotary(odd, swapped, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    for a, b in zip(got, want):  # other kernels may sum in another order: one rounding
        assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())


def test_qk_extreme_rows():
    """A zero row stays zero (eps keeps it finite), an infinite one gives NaN
    there alone, and its neighbours are untouched."""
    q, k, cos, sin, pos, _, _, _ = qk_case((1, 4, 2, 1, 64, 64, False, "none"), torch.float32)
    q = q.clone()
    q[0, 1, 0] = 0
    q[0, 2, 1, 5] = float("inf")
    y, _ = fa.qk_norm_rotary(q, k, cos, sin, positions=pos)
    assert bool((y[0, 1, 0] == 0).all())
    assert bool(y[0, 2, 1].isnan().any())
    ok = torch.ones(4, 2, dtype=torch.bool, device="cuda")
    ok[2, 1] = False
    assert bool(y[0][ok].isfinite().all())


def test_qk_empty_and_graph_capture_and_streams():
    q = torch.empty(2, 0, 4, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    cos, sin = tables(8, 64)
    y, z = fa.qk_norm_rotary(q, q[:, :, :2], cos, sin, q_weight=w, k_weight=w)
    assert y.shape == (2, 0, 4, 64) and z.shape == (2, 0, 2, 64)
    (y.sum() + z.sum()).backward()
    assert bool((w.grad == 0).all())
    q, k, cos, sin, pos, ws, _, _ = qk_case(QK[1], torch.bfloat16)
    want = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_qk_weight_gradient_is_the_same_bits_every_time():
    q, k, cos, sin, pos, ws, gs, inter = qk_case((2, 701, 4, 2, 64, 64, False, "dim"),
                                                 torch.float32)
    ws = [w.requires_grad_(True) for w in ws]
    runs = []
    for _ in range(3):
        out = fa.qk_norm_rotary(q, k, cos, sin, q_weight=ws[0], k_weight=ws[1], positions=pos)
        runs.append(torch.autograd.grad(out, ws, gs))
    for r in runs[1:]:
        assert torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1])


# --------------------------------------------------------------------------- #
# orthogonalised updates
# --------------------------------------------------------------------------- #

def plain_ns(x, steps=5, coefficients=NEWTON_SCHULZ):
    """float64; (..., m, n)."""
    x = x.double()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(norm > 0, x / norm, torch.zeros_like(x))
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    cs = coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    for a, b, c in cs:
        g = x @ x.mT
        x = a * x + (b * g + c * g @ g) @ x
    return x.mT if tall else x


def gradient(shape, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    m, n = shape[-2:]
    if kind == "spiky":
        r = max(1, min(m, n) // 16)
        x = x + 30 * (torch.randn(*shape[:-1], r, generator=g, device="cuda")
                      @ torch.randn(*shape[:-2], r, n, generator=g, device="cuda"))
    return 1e-3 * x


# relative 2-norm error allowed: the products' error (bfloat16: float16 operands,
# 2^-12 each with the identity and diagonals kept apart, times the slope of five
# steps; the others: float32-like) and the output's rounding
NS_TOL = {torch.float32: 2e-5, torch.float16: 3e-4, torch.bfloat16: 2.5e-3}

NS_SHAPES = [(1, 1), (1, 7), (5, 1), (16, 16), (33, 20), (64, 64), (65, 130), (127, 129),
             (128, 128), (200, 72), (257, 300), (384, 1000), (1000, 384), (640, 640)]


def rel(got, want):
    d = torch.linalg.vector_norm(got.double() - want)
    return float(d / torch.linalg.vector_norm(want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["noise", "spiky"])
@pytest.mark.parametrize("shape", NS_SHAPES)
def test_orthogonalize(shape, kind, dtype):
    x = gradient(shape, kind).to(dtype)
    y = fa.orthogonalize(x)
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    assert rel(y, plain_ns(x)) < NS_TOL[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
def test_orthogonalize_singular_values_follow_the_polynomial(dtype):
    u = torch.linalg.qr(torch.randn(48, 48, dtype=torch.float64, device="cuda"))[0]
    v = torch.linalg.qr(torch.randn(90, 48, dtype=torch.float64, device="cuda"))[0]
    s = torch.logspace(0, -2, 48, dtype=torch.float64, device="cuda")
    x = ((u * s) @ v.mT).to(dtype)
    got = torch.linalg.svdvals(fa.orthogonalize(x).double())
    assert float(got.max()) < 1.25 and float(got.min()) > 0.6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 40, 56), (2, 3, 130, 70), (150, 12, 20), (5, 200, 333)])
def test_orthogonalize_stacks(shape, dtype):
    x = gradient(shape, "noise", seed=2).to(dtype)
    y = fa.orthogonalize(x)
    want = plain_ns(x)
    assert y.shape == x.shape
    worst = max(rel(a, b) for a, b in zip(y.flatten(0, -3), want.flatten(0, -3)))
    assert worst < NS_TOL[dtype]
    # a matrix of a stack is what it is alone
    one = fa.orthogonalize(x.flatten(0, -3)[1])
    assert rel(one, y.flatten(0, -3)[1].double()) < NS_TOL[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
def test_orthogonalize_scale_does_not_matter(dtype):
    x = gradient((72, 100), "noise", seed=3)
    want = fa.orthogonalize(x.to(dtype))
    for e in ((-20, 10) if dtype == torch.float16 else (-100, 60)):
        # powers of two scale float16 exactly only above its subnormals
        got = fa.orthogonalize((x * 2.0 ** (10 + e if dtype == torch.float16 and e < 0 else e)).to(dtype))
        if dtype != torch.float16:
            assert torch.equal(got, want)
        else:
            assert bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(24, 40), (300, 260)])
def test_orthogonalize_zero_nan_and_inf(size, dtype):
    x = gradient((4, *size), "noise", seed=4).to(dtype)
    clean = fa.orthogonalize(x)
    x[0] = 0
    x[1, 3, 5] = float("nan")
    x[2, size[0] - 1, 0] = -float("inf")
    y = fa.orthogonalize(x)
    assert bool((y[0] == 0).all())
    assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
    assert torch.equal(y[3], clean[3])


def test_orthogonalize_views_strides_steps_and_coefficients():
    base = gradient((6, 90, 70), "noise", seed=5)
    want = plain_ns(base[::2, 5:75, 3:53].contiguous())
    for dtype in (torch.float32, torch.bfloat16):
        b = base.to(dtype)
        v = b[::2, 5:75, 3:53]
        assert rel(fa.orthogonalize(v), plain_ns(v)) < NS_TOL[dtype]
        assert rel(fa.orthogonalize(v.mT), plain_ns(v).mT) < NS_TOL[dtype]
        e = v[0].expand(3, 70, 50)
        assert rel(fa.orthogonalize(e), plain_ns(e)) < NS_TOL[dtype]
    x = base[0]
    for steps in (1, 2, 3, 8):
        assert rel(fa.orthogonalize(x, steps=steps), plain_ns(x, steps)) < NS_TOL[torch.float32]
    many = [(4.0, -6.0, 2.5), (3.0, -4.0, 1.8), (1.875, -1.25, 0.375)]
    assert rel(fa.orthogonalize(x, steps=3, coefficients=many), plain_ns(x, 3, many)) < 2e-5
    cubic = (1.5, -0.5, 0.0)
    assert rel(fa.orthogonalize(x, steps=10, coefficients=cubic), plain_ns(x, 10, cubic)) < 2e-5
    assert want.shape == (3, 70, 50)


def test_orthogonalize_empty():
    for shape in ((0, 5, 5), (3, 0, 4), (4, 0)):
        assert fa.orthogonalize(torch.empty(shape, device="cuda")).shape == shape


def test_orthogonalize_same_bits_every_time_and_in_a_graph():
    x = gradient((2, 300, 500), "spiky", seed=6).to(torch.bfloat16)
    a = fa.orthogonalize(x)
    for _ in range(3):
        assert torch.equal(fa.orthogonalize(x), a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = fa.orthogonalize(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def plain_muon(w, g, m, lr, mu, nesterov, wd, scale):
    w, g, m = w.double(), g.double(), m.double()
    m = mu * m + g
    u = g + mu * m if nesterov else m
    rows, cols = w.shape[0], w[0].numel()
    s = {"aspect": math.sqrt(max(1, rows / cols)), "rms": 0.2 * math.sqrt(max(rows, cols)),
         "none": 1.0}[scale]
    return (1 - lr * wd) * w - lr * s * plain_ns(u.reshape(rows, cols)).view(w.shape), m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nesterov,wd,scale", [(True, 0.0, "aspect"), (False, 0.1, "rms"),
                                               (True, 0.01, "none")])
def test_muon_step(dtype, nesterov, wd, scale):
    shapes = [(64, 96), (96, 64), (64, 96), (16, 3, 3, 3), (130, 50), (1, 9), (300, 280)]
    g = torch.Generator(device="cuda").manual_seed(7)
    W = [(torch.randn(s, generator=g, device="cuda") / 8).to(dtype) for s in shapes]
    G = [(1e-2 * torch.randn(s, generator=g, device="cuda")).to(dtype) for s in shapes]
    M = [1e-2 * torch.randn(s, generator=g, device="cuda") for s in shapes]
    want = [plain_muon(w, gr, m, 0.02, 0.9, nesterov, wd, scale) for w, gr, m in zip(W, G, M)]
    fa.muon_step(W, G, M, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=wd, scale=scale)
    for w, m, (ww, wm) in zip(W, M, want):
        assert rel(m, wm) < 2.0 ** -22
        # one rounding of the weight, and the update's own error times its share of the weight
        tol = 2 * U[dtype] + NS_TOL[dtype] * 0.02 * 0.2 * 20 / float(ww.square().mean().sqrt()) / 8
        assert rel(w, ww) < tol


def test_muon_optimizer_matches_the_functional_step_and_survives_checkpoints():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 24, 3), torch.nn.Conv2d(24, 8, 3)).cuda()
    net = net.to(memory_format=torch.channels_last)
    ps = [p for p in net.parameters() if p.dim() > 1]
    opt = fa.Muon(ps, lr=0.05, weight_decay=0.1)
    twins = [p.detach().clone(memory_format=torch.preserve_format) for p in ps]
    moms = [torch.zeros_like(t) for t in twins]
    x = torch.randn(2, 3, 20, 20, device="cuda").to(memory_format=torch.channels_last)
    for _ in range(3):
        opt.zero_grad()
        net(x).square().mean().backward()
        grads = [p.grad.clone(memory_format=torch.preserve_format) for p in ps]
        opt.step()
        fa.muon_step(twins, grads, moms, lr=0.05, weight_decay=0.1)
    for p, t, g in zip(ps, twins, grads):
        assert torch.equal(p.detach(), t)
    half = [torch.nn.Parameter(t.to(torch.bfloat16)) for t in twins]
    o1 = fa.Muon(half, lr=0.01)
    for h in half:
        h.grad = torch.randn_like(h)
    o1.step()
    copies = [torch.nn.Parameter(h.detach().clone(memory_format=torch.preserve_format)) for h in half]
    o2 = fa.Muon(copies, lr=0.01)
    o2.load_state_dict(o1.state_dict())
    for h, c in zip(half, copies):
        assert o2.state[c]["momentum_buffer"].dtype == torch.float32
        h.grad = torch.randn_like(h)
        c.grad = h.grad.clone(memory_format=torch.preserve_format)
    o1.step()
    o2.step()
    for h, c in zip(half, copies):
        assert torch.equal(h, c)


def test_muon_orders_of_memory():
    """A channels-last kernel is updated as its contiguous twin is, whatever the
    gradient's layout."""
    g = torch.Generator(device="cuda").manual_seed(9)
    w = torch.randn(12, 5, 3, 3, generator=g, device="cuda")
    gr = torch.randn(12, 5, 3, 3, generator=g, device="cuda")
    m = torch.zeros_like(w)
    want, _ = plain_muon(w, gr, m, 0.1, 0.95, True, 0.0, "aspect")
    cl = torch.channels_last
    for wf in (torch.contiguous_format, cl):
        for gf in (torch.contiguous_format, cl):
            w1 = w.clone().contiguous(memory_format=wf)
            m1 = torch.zeros_like(w1)
            fa.muon_step([w1], [gr.contiguous(memory_format=gf)], [m1], lr=0.1)
            assert rel(w1, want) < 2e-6
            assert torch.equal(m1, gr)


# --------------------------------------------------------------------------- #
# the product kernel's other shapes: K in parts, pairs of blocks, many shapes
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(64, 5000), (5000, 64), (100, 3501), (2, 130, 2050),
                                   (2050, 190), (3, 20, 1999)])
def test_orthogonalize_long_and_narrow(shape, dtype):
    """Few tiles: K is split over blocks and joined."""
    x = gradient(shape, "noise", seed=11).to(dtype)
    y = fa.orthogonalize(x)
    assert rel(y, plain_ns(x)) < NS_TOL[dtype]
    assert torch.equal(fa.orthogonalize(x), y)  # joined in one order


@pytest.mark.parametrize("shape", [(20, 1030, 1100), (5, 2100, 1500), (4100, 4200)])
def test_orthogonalize_large(shape):
    """Many tiles: pairs of blocks share them; sizes that leave a block of the
    last pair without rows."""
    x = gradient(shape, "spiky", seed=12).to(torch.bfloat16)
    y = fa.orthogonalize(x)
    want = plain_ns(x)
    worst = max(rel(a, b) for a, b in zip(y.view(-1, *shape[-2:]), want.view(-1, *shape[-2:])))
    assert worst < NS_TOL[torch.bfloat16]
    assert torch.equal(fa.orthogonalize(x), y)


def test_orthogonalize_float32_large():
    x = gradient((2, 1100, 1290), "spiky", seed=13)
    assert max(rel(a, b) for a, b in zip(fa.orthogonalize(x), plain_ns(x))) < NS_TOL[torch.float32]


def test_muon_step_with_more_shapes_than_a_launch_holds():
    g = torch.Generator(device="cuda").manual_seed(14)
    shapes = [(8 + 7 * i, 90 - 5 * i) for i in range(13)] * 2 + [(33, 20)] * 120
    W = [torch.randn(s, generator=g, device="cuda") for s in shapes]
    G = [torch.randn(s, generator=g, device="cuda") for s in shapes]
    M = [torch.randn(s, generator=g, device="cuda") for s in shapes]
    want = [plain_muon(w, gr, m, 0.1, 0.95, True, 0.0, "none") for w, gr, m in zip(W, G, M)]
    fa.muon_step(W, G, M, lr=0.1, scale="none")
    for w, m, (ww, wm) in zip(W, M, want):
        assert rel(w, ww) < 2e-6 and rel(m, wm) < 2.0 ** -22


def test_orthogonalize_on_two_streams_at_once():
    xs = [gradient((3, 300, 420), "noise", seed=20 + i).to(torch.bfloat16) for i in range(2)]
    want = [fa.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fa.orthogonalize(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_in_place_outputs_count_as_modified():
    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    loss = (w * w).sum()
    with torch.no_grad():
        fa.muon_step([w], [torch.randn_like(w)], [torch.zeros_like(w)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_training_example_learns():
    import sys

    from conftest import REPO
    sys.path.insert(0, str(REPO / "examples"))
    import train_restoration

    losses = train_restoration.train(steps=40, size=64, frames=4)
    assert all(math.isfinite(v) for v in losses)
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5]), (losses[:5], losses[-5:])


@pytest.mark.parametrize("shape,dtype", [((4100, 4200), torch.bfloat16), ((1500, 1400), torch.float32)])
def test_a_launch_may_last_longer_than_the_limit_of_its_waits(shape, dtype):
    """32 steps on 4100 x 4200 take about 10 ms, a tile below 0.1 ms: a limit of
    3 ms for each wait is never reached.  (That shape runs in pairs of blocks.)"""
    from frame_analytics_b200 import _cabi
    L = _cabi.load()
    x = gradient(shape, "noise", seed=15).to(dtype)
    cubic = (1.5, -0.5, 0.0)
    want = fa.orthogonalize(x, steps=32, coefficients=cubic)
    t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    assert L.fa_b200_orthogonalize_wait_limit(3_000_000) == 0
    try:
        t[0].record()
        got = fa.orthogonalize(x, steps=32, coefficients=cubic)
        t[1].record()
        torch.cuda.synchronize()
        fa.orthogonalize(x[:8, :8])  # a wait that gave up would be reported here
    finally:
        assert L.fa_b200_orthogonalize_wait_limit(0) == 0
    if dtype == torch.bfloat16:
        assert t[0].elapsed_time(t[1]) > 2 * 3
    assert torch.equal(got, want)


def test_lists_that_one_workspace_does_not_hold():
    """45 x 2048 x 2048 would take 2.3 GB, 12 x (2048 x 4096 and 4096 x 4096)
    3.4 GB: they run in parts that share 2 GiB.  Matrices on either side of a
    cut against float64."""
    x = gradient((45, 2048, 2048), "noise", seed=16).to(torch.bfloat16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = fa.orthogonalize(x)
    extra = torch.cuda.max_memory_allocated() - before - y.numel() * y.element_size()
    assert extra <= (2 << 30) + (64 << 20)
    for i in (0, 1, 21, 41, 42, 43, 44):
        assert rel(y[i], plain_ns(x[i])) < NS_TOL[torch.bfloat16]
    del x, y
    shapes = [(2048, 4096), (4096, 4096)] * 12
    g = torch.Generator(device="cuda").manual_seed(17)
    W = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in shapes]
    G = [torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in shapes]
    M = [torch.zeros(s, device="cuda") for s in shapes]
    fa.muon_step(W, G, M, lr=1.0, scale="none", nesterov=False)
    for i in (0, 1, 13, 14, 15, 16, 23):
        assert torch.equal(M[i], G[i].float())
        assert rel(W[i], -plain_ns(G[i])) < NS_TOL[torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_small_matrix_is_updated_alike_whatever_the_list_holds(dtype):
    """Matrices up to 64 x 128 run in float32, alone, beside larger ones, and on
    either side of a cut at 128 matrices or 8 shapes."""
    g = torch.Generator(device="cuda").manual_seed(18)

    def step(shapes, at):
        G = [grads[s] for s in shapes]
        W = [torch.zeros(s, dtype=dtype, device="cuda") for s in shapes]
        M = [torch.zeros(s, device="cuda") for s in shapes]
        fa.muon_step(W, G, M, lr=1.0, scale="none", nesterov=False)
        for s, w in zip(shapes, W):
            assert rel(w, -plain_ns(grads[s])) < NS_TOL[dtype]
        return [W[i] for i in at]

    small = [(64, 64), (16, 27), (128, 64), (1, 5), (64, 128), (9, 100), (33, 20), (40, 40), (7, 7),
             (12, 80)]
    large = [(300, 280), (65, 64), (64, 129)]
    grads = {s: torch.randn(s, generator=g, device="cuda").to(dtype) for s in small + large}
    alone = {s: step([s], [0])[0] for s in small}
    for s in small:  # float32 and one rounding of the output
        assert rel(alone[s], -plain_ns(grads[s])) < 2 * U[dtype] + 2e-5
    mixed = [large[0]] + small + large[1:] + small[::-1]
    at = [i for i, s in enumerate(mixed) if s in small]
    for i, w in zip(at, step(mixed, at)):
        assert torch.equal(w, alone[mixed[i]])
    many = [small[i % 10] for i in range(150)] + [large[0]]
    for i, w in enumerate(step(many, range(150))):
        assert torch.equal(w, alone[many[i]])


def test_mixed_lists_in_a_graph_and_on_two_streams():
    """Small matrices run beside the larger ones: what follows on the caller's
    stream waits for both."""
    g = torch.Generator(device="cuda").manual_seed(19)
    shapes = [(64, 64), (300, 280), (16, 27), (128, 64), (65, 200)]
    G = [torch.randn(s, generator=g, device="cuda") for s in shapes]

    def step(x):
        W = [torch.zeros_like(t) for t in x]
        fa.muon_step(W, x, [torch.zeros_like(t) for t in x], lr=1.0, nesterov=False)
        return [2 * w for w in W]

    want = step(G)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step([t.clone() for t in G]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got.append(step(G))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for run in got:
        assert all(torch.equal(a, b) for a, b in zip(run, want))


@pytest.mark.parametrize("relaid", ["checkpoint", "in place"])
@pytest.mark.parametrize("frm,to", [(torch.contiguous_format, torch.channels_last),
                                    (torch.channels_last, torch.contiguous_format)])
def test_muon_momentum_follows_its_parameters_layout(frm, to, relaid):
    """Against a run that keeps its layout: the momenta are the same numbers, the
    weights differ by what two sums in other orders may (each within NS_TOL of
    the update, whose norm is at most 1.3 sqrt(cols) lr)."""
    g = torch.Generator(device="cuda").manual_seed(21)
    w = torch.randn(24, 12, 3, 3, generator=g, device="cuda") / 8
    grads = [torch.randn(w.shape, generator=g, device="cuda") for _ in range(3)]

    def optimizer(start, fmt):
        p = torch.nn.Parameter(start.detach().clone().contiguous(memory_format=fmt))
        return p, fa.Muon([p], lr=0.05)

    def advance(p, opt, gr):
        p.grad = gr.contiguous(memory_format=torch.contiguous_format).clone()
        opt.step()

    keep, kept = optimizer(w, frm)
    p, opt = optimizer(w, frm)
    advance(keep, kept, grads[0])
    advance(p, opt, grads[0])
    assert torch.equal(p, keep)
    if relaid == "checkpoint":
        saved = opt.state_dict()
        p, opt = optimizer(p, to)
        opt.load_state_dict(saved)
    else:
        p.data = p.data.contiguous(memory_format=to)
    for gr in grads[1:]:
        advance(keep, kept, gr)
        advance(p, opt, gr)
    assert p.is_contiguous(memory_format=to)
    m = opt.state[p]["momentum_buffer"]
    assert m.stride() == p.stride() and torch.equal(m, kept.state[keep]["momentum_buffer"])
    update = 2 * 1.3 * math.sqrt(24) * 0.05
    tol = 2 * NS_TOL[torch.float32] * update + 2 * 2 * U[torch.float32] * float(w.norm())
    assert float((p - keep).detach().norm()) < tol


def test_muon_takes_any_layout():
    g = torch.Generator(device="cuda").manual_seed(22)
    w = torch.randn(40, 72, generator=g, device="cuda") / 8
    gr = torch.randn(40, 72, generator=g, device="cuda")
    m = torch.randn(40, 72, generator=g, device="cuda")

    def layouts(t):
        wide = [torch.full((40, 150), 7.0, device="cuda") for _ in range(2)]
        return [t.clone(), t.t().contiguous().t(), wide[0][:, 3:147:2].copy_(t),
                wide[1][:, 150 - 72:].copy_(t)]

    want_w, want_m = w.clone(), m.clone()
    fa.muon_step([want_w], [gr], [want_m], lr=0.1)
    for i in range(3):
        for j in range(3):
            for k in range(3):
                wl, gl, ml = layouts(w)[i], layouts(gr)[j], layouts(m)[k]
                fa.muon_step([wl], [gl], [ml], lr=0.1)
                assert torch.equal(wl, want_w) and torch.equal(ml, want_m) and torch.equal(gl, gr)
    sliced = layouts(w)[3]
    base = sliced._base
    fa.muon_step([sliced], [gr], [m.clone()], lr=0.1)
    assert torch.equal(sliced, want_w) and bool((base[:, :3] == 7).all())
    # 3-D kernels, channels last
    w5, g5 = (torch.randn(8, 4, 3, 2, 2, generator=g, device="cuda") for _ in range(2))
    last = w5.contiguous(memory_format=torch.channels_last_3d)
    m5 = torch.zeros_like(last)
    fa.muon_step([w5], [g5], [torch.zeros_like(w5)], lr=0.1)
    fa.muon_step([last], [g5], [m5], lr=0.1)
    assert torch.equal(last, w5) and torch.equal(m5, g5)
    # one row, spread over the list's rows
    shared = torch.zeros(1, 72, device="cuda").expand(40, 72)
    for args in (([shared], [gr], [m]), ([w], [gr], [shared])):
        with pytest.raises(ValueError, match="share memory"):
            fa.muon_step(*args, lr=0.1)
    fa.muon_step([w.clone()], [gr[:1].expand(40, 72)], [m], lr=0.1)


def test_muon_refuses_a_checkpoint_of_another_shape():
    a, b = (torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in ((4, 6), (1, 6)))
    one, two = fa.Muon([a]), fa.Muon([b])
    b.grad = torch.ones_like(b)
    two.step()
    with pytest.raises(ValueError, match="shape"):
        one.load_state_dict(two.state_dict())


def test_muon_refuses_gradients_that_it_would_overwrite():
    a, b = (torch.randn(300, 280, device="cuda") for _ in range(2))
    m, n = torch.zeros_like(a), torch.zeros_like(a)
    before = [t.clone() for t in (a, b, m, n)]
    for ws, gs, ms in (([a], [m], [m]), ([a, b], [n, m], [m, n]), ([a, b], [b, a], [m, n]),
                       ([a, a], [b, b], [m, n]), ([a, b], [b, b], [m, m])):
        with pytest.raises(ValueError):
            fa.muon_step(ws, gs, ms, lr=0.1)
    assert all(torch.equal(x, y) for x, y in zip((a, b, m, n), before))
    # its own weight is read before it is written
    want, _ = plain_muon(a, a, m, 0.1, 0.95, True, 0.0, "none")
    fa.muon_step([a], [a], [m], lr=0.1, scale="none")
    assert rel(a, want) < 2e-6 and torch.equal(m, before[0])


def test_qk_out_refuses_shared_memory():
    q = torch.randn(2, 6, 4, 64, device="cuda")
    k = torch.randn(2, 6, 4, 64, device="cuda")
    o, p = torch.empty_like(q), torch.empty_like(k)
    turned = q.view(2, 4, 6, 64).transpose(1, 2)  # q's memory in another order
    before = q.clone(), k.clone()
    for a, b, out in ((q, k, (o, o)), (q, k, (k, p)), (q, k, (o, q)), (q, k, (k, q)),
                      (q, q, (q, p)), (q, q, (o, q)), (q, k, (turned, p)), (k, q, (o, turned))):
        with pytest.raises(ValueError, match="share memory"):
            fa.qk_norm_rotary(a, b, out=out)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    want = fa.qk_norm_rotary(q, k)
    packed = torch.cat((q, k), 2)
    a, b = packed[:, :, :4], packed[:, :, 4:]
    got = fa.qk_norm_rotary(a, b, out=(a, b))  # both in place, interleaved in one buffer
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    same = fa.qk_norm_rotary(q, q, out=(o, p))  # one input twice
    assert torch.equal(same[0], want[0]) and torch.equal(same[1], want[0])


def test_graphs_of_a_training_pass_replay_in_any_order():
    """A workspace made under capture is zeroed by that graph's replays alone:
    it must not serve another graph, nor a graph the buffer of eager calls."""
    from frame_analytics_b200 import backend
    q, k, cos, sin, pos, ws, gs, _ = qk_case((2, 65, 4, 2, 64, 64, False, "dim"), torch.float32)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *ws)]

    def backward():
        out = fa.qk_norm_rotary(leaves[0], leaves[1], cos, sin, q_weight=leaves[2],
                                k_weight=leaves[3], positions=pos)
        return torch.autograd.grad(out, leaves, gs)

    want = backward()
    stream = torch.cuda.Stream()
    backend._ws.pop((0, stream.cuda_stream), None)  # as on a stream that has run nothing
    torch.cuda.synchronize()
    graphs, got = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            got.append(backward())
    kept = backend._ws.get((0, stream.cuda_stream))
    if kept is not None:  # what memory that nothing has zeroed may hold
        kept.fill_(0x55)
    for i in (1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(got[i], want):
            assert torch.equal(a, b)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        backward()  # the stream has a buffer now
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        again = backward()
    backend._ws.pop((0, stream.cuda_stream)).fill_(0x55)  # and gives it up
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_muon_refuses_strided_tensors_given_twice():
    a, b = (torch.randn(9, 8, device="cuda").t() for _ in range(2))
    g, m, n = (torch.zeros(8, 9, device="cuda") for _ in range(3))
    before = a.clone()
    for ws, ms in (([a, a], [m, n]), ([a, b], [b, m]), ([g, n], [a, a]), ([a, g], [m, a])):
        with pytest.raises(ValueError, match="twice"):
            fa.muon_step(ws, [torch.ones_like(w) for w in ws], ms, lr=0.1)
    assert torch.equal(a, before) and bool((m == 0).all())
