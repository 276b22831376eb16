"""The 8-bit block operators on the GPU, against plain float64 formulas.

Tolerances: u is half a step of the output's type relative to a value (2^-24,
2^-11, 2^-8 for float32, float16, bfloat16); each output is rounded once.  Behind
it stand float32 sums: a thread adds at most n / 32 + 64 terms of a row of n one
after the other, then a few levels of a tree, so a row's mean, variance and dot
products are off by at most (n / 32 + 80) 2^-24 of the sum of their terms'
magnitudes.  Packed values are compared bit for bit.
"""

from __future__ import annotations

import math
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F

import frame_analytics_b200 as fa

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rand(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def within(got, want, tol, dtype):
    err = (got.double() - want).abs()
    tol = tol + TINY[dtype]
    assert bool((err <= tol).all()), (err / tol).max().item()


# --------------------------------------------------------------------------- #
# packing
# --------------------------------------------------------------------------- #

def plain_pack(x):
    """(values in x's dtype, codes) from the definition, group by group, float64."""
    dtype, width = x.dtype, x.shape[-1]
    rows = x.reshape(-1, width)
    values, codes = torch.empty_like(rows), torch.zeros(
        rows.shape[0], -(-width // 64) * 64, dtype=torch.uint8, device=x.device)
    most = torch.finfo(dtype).max
    for c in range(0, width, 64):
        v = rows[:, c:c + 64].double()
        lo, hi = v.amin(1, keepdim=True), v.amax(1, keepdim=True)
        d = (hi - lo).float()
        fine = d.isfinite()
        d = torch.where(fine, d, torch.zeros_like(d)).double()
        e = torch.full_like(d, -126)
        for _ in range(300):  # the smallest e with d <= 255 2^e
            e = torch.where(d > 255 * torch.exp2(e), e + 1, e)
        s = torch.exp2(e)
        q = ((v - lo).float().double() / s).round()
        top = (d / s).round()
        over = ((top * s + lo).to(dtype).double().abs() > most)
        q = torch.where(over, torch.minimum(q, top - 1), q)
        values[:, c:c + 64] = torch.where(fine, (q * s + lo).to(dtype).double(), math.nan).to(dtype)
        codes[:, c:c + v.shape[1]] = torch.where(fine, q, torch.zeros_like(q)).to(torch.uint8)
    return values.view(x.shape), codes.view(*x.shape[:-1], -1)


def same_bits(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(
        a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) or (
        torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)))


KINDS = {
    "normal": lambda x: x,
    "offset": lambda x: x + 1000,
    "wide": lambda x: x * torch.exp2(torch.arange(x.shape[-1], device=x.device) % 40 - 20.0),
    "one-sided": lambda x: x.relu(),
    "constant": lambda x: torch.full_like(x, 0.37),
    "zero": lambda x: torch.zeros_like(x),
    "whole": lambda x: (x * 90).round(),
    "halves": lambda x: (x * 200).round() / 2,      # ties between codes
    "tiny": lambda x: x * 2.0 ** -136,
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 64), (4, 65), (3, 200), (5, 128),
                                   (33, 1000), (1000,), (130, 8)])
def test_pack_bit_for_bit(shape, kind, dtype):
    x = KINDS[kind](rand(*shape, seed=1)).to(dtype)
    want, codes = plain_pack(x)
    p = fa.pack8(x)
    assert p.shape == x.shape and p.dtype == dtype
    assert torch.equal(p.codes, codes)
    assert same_bits(fa.unpack8(p), want + 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_is_within_its_bound(dtype):
    x = rand(64, 640, seed=2, scale=3.0, dtype=dtype)
    back = fa.unpack8(fa.pack8(x))
    v = x.double().view(64, 10, 64)
    d = v.amax(-1, keepdim=True) - v.amin(-1, keepdim=True)
    err = (back.double().view_as(v) - v).abs()
    # s / 2 < d / 255, and the value's own rounding
    assert bool((err <= d / 255 + U[dtype] * (v.abs() + d / 255)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_of_the_largest_and_of_what_is_not_finite(dtype):
    most = torch.finfo(dtype).max
    x = rand(12, 192, seed=3).to(dtype)
    x[0, 3] = math.inf
    x[1, 70] = -math.inf
    x[2, 191] = math.nan
    x[3, 5], x[3, 6] = math.inf, -math.inf
    x[4] = most
    x[5] = -most
    x[6, 0] = most
    x[7, 9], x[7, 10] = most, -most           # a spread past float32 for two of the types
    x[8, 100] = -most
    x[9, 0], x[9, 1] = most, most / 2
    x[10] = math.nan
    x[11] = math.inf
    want, _ = plain_pack(x)
    got = fa.unpack8(fa.pack8(x))
    assert same_bits(got, want)
    assert bool(got[0, :64].isnan().all()) and bool(got[0, 64:].isfinite().all())
    assert bool((got[4] == most).all()) and bool(got[6].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("view", [
    lambda x: x.mT, lambda x: x[:, 1:], lambda x: x[::3], lambda x: x[:, :100],
    lambda x: x[:, ::2], lambda x: x[0].expand(9, -1), lambda x: x[:, :1].expand(-1, 70),
    lambda x: x.view(4, 10, 136).transpose(0, 1), lambda x: x[3:, 8:72],
])
def test_pack_of_views(view, dtype):
    x = view(rand(40, 136, seed=4, dtype=dtype))
    want, codes = plain_pack(x.contiguous())
    p = fa.pack8(x)
    assert torch.equal(p.codes, codes) and same_bits(fa.unpack8(p), want)


def test_unpack_of_what_was_moved():
    x = rand(6, 200, seed=5, dtype=torch.bfloat16)
    p = fa.pack8(x)
    want = fa.unpack8(p)
    host = p._replace(codes=p.codes.cpu(), ranges=p.ranges.cpu())
    back = host._replace(codes=host.codes.cuda(), ranges=host.ranges.cuda())
    assert torch.equal(fa.unpack8(back), want)
    at = torch.empty(p.codes.numel() + 5, dtype=torch.uint8, device="cuda")[5:].view(p.codes.shape)
    rt = torch.empty(p.ranges.numel() + 1, dtype=torch.int32, device="cuda")[1:].view(p.ranges.shape)
    odd = p._replace(codes=at.copy_(p.codes), ranges=rt.copy_(p.ranges))  # odd addresses
    assert torch.equal(fa.unpack8(odd), want)
    with pytest.raises(TypeError):
        fa.unpack8(p._replace(codes=host.codes))


@pytest.mark.parametrize("width", [2112, 2111])
def test_pack_past_2_31_values(width):
    rows = (1 << 31) // width + 77
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-50:] = rand(50, width, seed=6).bfloat16()
    x[:50] = rand(50, width, seed=7).bfloat16()
    p = fa.pack8(x)
    back = fa.unpack8(p)
    for part in (slice(0, 60), slice(rows - 60, rows)):
        want, codes = plain_pack(x[part])
        assert torch.equal(p.codes[part], codes) and torch.equal(back[part], want)
    assert not bool(back[60:-60].any())


# --------------------------------------------------------------------------- #
# layer norm
# --------------------------------------------------------------------------- #

# leading shape, width, residual, affine, float32 weights
NORMS = [
    ((1,), 1, False, "none", False),
    ((2,), 3, True, "both", False),
    ((1,), 1024, True, "both", False),
    ((4, 5), 64, False, "both", False),
    ((37,), 577, False, "both", True),
    ((130,), 200, True, "weight", False),
    ((3, 3), 192, True, "both", True),
    ((300,), 256, False, "bias", False),
    ((65,), 512, True, "both", False),
    ((21,), 1000, True, "none", False),
    ((19,), 1025, False, "both", False),
    ((9,), 2048, True, "both", True),
    ((5,), 2056, False, "both", False),
    ((7,), 4096, True, "both", False),
    ((3,), 8192, False, "both", False),
    ((2,), 8200, True, "both", False),
    ((3,), 12001, False, "both", False),
    ((2,), 40000, True, "both", True),
    ((2000,), 72, True, "both", False),
]


def norm_case(case, dtype, seed=0):
    lead, n, residual, affine, wide = case
    wt = torch.float32 if wide else dtype
    x = (rand(*lead, n, seed=seed) * 2 + 0.5).to(dtype)
    res = rand(*lead, n, seed=seed + 1, dtype=dtype) if residual else None
    w = (1 + 0.3 * rand(n, seed=seed + 2)).to(wt) if affine in ("both", "weight") else None
    b = (0.3 * rand(n, seed=seed + 3)).to(wt) if affine in ("both", "bias") else None
    gy = rand(*lead, n, seed=seed + 4, dtype=dtype)
    gs = rand(*lead, n, seed=seed + 5, dtype=dtype) if residual else None
    return x, res, w, b, gy, gs


def norm_sum(x, res):
    return x if res is None else (x.double() + res.double()).to(x.dtype)


def norm_terms(s, eps):
    """float64 mean, 1 / deviation, and the relative error of either float32 sum."""
    s = s.double()
    n = s.shape[-1]
    m = s.mean(-1, keepdim=True)
    r = 1 / ((s - m).square().mean(-1, keepdim=True) + eps).sqrt()
    depth = n / 32 + 80
    em = E * depth * s.abs().mean(-1, keepdim=True)   # of the mean
    return m, r, em, E * depth


def check_norm(y, s, w, b, eps, dtype):
    m, r, em, rel = norm_terms(s, eps)
    w = 1.0 if w is None else w.double()
    b = torch.zeros((), device="cuda", dtype=torch.float64) if b is None else b.double()
    part = (s.double() - m) * r * w
    want = part + b
    # the mean's error moves the value and, squared, the variance
    tol = U[dtype] * want.abs() + (rel + 8 * E) * part.abs() + (em + E * s.double().abs()) * r * abs(w) \
        + E * b.abs()
    within(y, want, tol * 1.01 + part.abs() * (em * r) ** 2, dtype)


def check_norm_grad(got, s, kept, w, b, gy, gs, eps, dtype):
    """`kept`: what the backward pass has of s."""
    m, r, em, rel = norm_terms(s, eps)
    n = s.shape[-1]
    xh = (kept.double() - m) * r
    exh = (rel + 8 * E + (em * r) ** 2) * xh.abs() + (em + E * kept.double().abs()) * r
    dy = gy.double()
    wd = torch.ones(n, device="cuda", dtype=torch.float64) if w is None else w.double()
    g = dy * wd
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    e2 = rel * a2 + (g.abs() * exh).mean(-1, keepdim=True)
    dx = r * (g - c1 - xh * c2)
    tol = r * (rel * a1 + xh.abs() * e2 + exh * c2.abs()) \
        + (rel + 16 * E) * r * (g.abs() + a1 + xh.abs() * a2)
    if gs is not None:
        dx = dx + gs.double()
        tol = tol + 2 * E * gs.double().abs()
    within(got[0], dx, (1 + 2 * U[dtype]) * tol + U[dtype] * dx.abs(), dtype)
    i = 1
    if gs is not None:
        assert torch.equal(got[1], got[0])
        i = 2
    # sums over rows: a warp adds its rows one after the other, then parts in order
    rows = s.numel() // n
    over = tuple(range(s.dim() - 1))
    for p, term, err in ((w, dy * xh, dy.abs() * exh), (b, dy, torch.zeros_like(dy))):
        if p is None:
            continue
        want = term.sum(over)
        tol = E * (min(rows, 400) + 40) * term.abs().sum(over) + err.sum(over)
        within(got[i], want, (1 + 2 * U[p.dtype]) * tol + U[p.dtype] * want.abs(), p.dtype)
        assert got[i].dtype == p.dtype and got[i].shape == p.shape
        i += 1
    assert i == len(got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", NORMS)
def test_norm_forward(case, dtype):
    x, res, w, b, _, _ = norm_case(case, dtype)
    got = fa.layer_norm(x, w, b, residual=res, eps=1e-5)
    s = norm_sum(x, res)
    if res is not None:
        got, total = got
        assert torch.equal(total, s) and total.is_contiguous()
    assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
    check_norm(got, s, w, b, 1e-5, dtype)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", NORMS)
def test_norm_backward(case, dtype, keep8):
    x, res, w, b, gy, gs = norm_case(case, dtype, seed=10)
    leaves = [t.detach().requires_grad_(True) for t in (x, res, w, b) if t is not None]
    it = iter(leaves)
    xl, rl, wl, bl = (None if t is None else next(it) for t in (x, res, w, b))
    out = fa.layer_norm(xl, wl, bl, residual=rl, eps=1e-5, keep8=keep8)
    out = (out,) if res is None else out
    s = norm_sum(x, res)
    check_norm(out[0].detach(), s, w, b, 1e-5, dtype)
    got = torch.autograd.grad(out, leaves, (gy,) if res is None else (gy, gs))
    kept = fa.unpack8(fa.pack8(s)) if keep8 else s
    check_norm_grad(got, s, kept, w, b, gy, gs, 1e-5, dtype)


def test_norm_gradient_against_differences():
    x, res, w, b, gy, gs = norm_case(((3,), 11, True, "both", False), torch.float32, seed=20)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, res, w, b)]
    out = fa.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1], eps=1e-2)
    grads = torch.autograd.grad(out, leaves, (gy, gs))

    def value(ts):
        s = ts[0] + ts[1]
        y = F.layer_norm(s, (11,), ts[2], ts[3], 1e-2)
        return float((y * gy).sum() + (s * gs).sum())

    wide = [t.detach().double() for t in leaves]
    h = 1e-4
    for i in range(4):
        flat = wide[i].flatten()
        for j in range(0, flat.numel(), 3):
            vals = []
            for sign in (1, -1):
                moved = flat.clone()
                moved[j] += sign * h
                vals.append(value([*wide[:i], moved.view(wide[i].shape), *wide[i + 1:]]))
            fd = (vals[0] - vals[1]) / (2 * h)
            assert abs(fd - float(grads[i].flatten()[j])) < 2e-5 * (1 + abs(fd))


@pytest.mark.parametrize("width", [200, 1024, 8200])
def test_norm_of_an_offset_row_keeps_its_precision(width):
    x = rand(5, width, seed=21) + 1000.0
    check_norm(fa.layer_norm(x), x, None, None, 1e-5, torch.float32)
    leaf = x.clone().requires_grad_(True)
    gy = rand(5, width, seed=22)
    w = torch.ones(width, device="cuda", requires_grad=True)
    got = torch.autograd.grad(fa.layer_norm(leaf, w, keep8=True), (leaf, w), gy)
    check_norm_grad(got, x, fa.unpack8(fa.pack8(x)), w.detach(), None, gy, None, 1e-5, torch.float32)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("width", [72, 1000, 9000])
def test_norm_rows_with_an_infinity_or_a_nan_stay_alone(width, keep8):
    x = rand(40, width, seed=23, dtype=torch.bfloat16)
    x[3, 5], x[17, 0] = math.inf, math.nan
    x[20] = 7.0                                  # no spread at all
    leaf = x.clone().requires_grad_(True)
    y = fa.layer_norm(leaf, keep8=keep8)
    dx, = torch.autograd.grad(y, leaf, rand(40, width, seed=24, dtype=torch.bfloat16))
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 17]] = True
    for t in (y, dx):
        assert bool(t[bad].isnan().any(-1).all()) and bool(t[~bad].isfinite().all())
    assert not bool(y[20].any())


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("view", [
    lambda t: t.mT, lambda t: t[:, 1:], lambda t: t[::3], lambda t: t[:, 8:136], lambda t: t[:, ::2],
    lambda t: t.view(4, 34, 136).transpose(0, 1),
])
def test_norm_of_views_and_of_expanded_gradients(view, keep8):
    x, res = rand(136, 136, seed=25), rand(136, 136, seed=26)
    a, b = view(x), view(res)
    w = 1 + 0.1 * rand(a.shape[-1] * 2, seed=27)[::2]
    leaves = [t.detach().requires_grad_(True) for t in (a, b, w)]
    y, s = fa.layer_norm(leaves[0], leaves[2], residual=leaves[1], keep8=keep8)
    want_s = a + b
    assert torch.equal(s, want_s)
    got = torch.autograd.grad((y.sum() + (3 * s).sum()), leaves)
    one = torch.ones_like(want_s)
    kept = fa.unpack8(fa.pack8(want_s)) if keep8 else want_s
    check_norm_grad(got, want_s, kept, w, None, one, 3 * one, 1e-5, torch.float32)


def test_norm_gradients_of_one_output_alone_and_of_an_operand_twice():
    x, res, w, b, gy, gs = norm_case(NORMS[8], torch.float32, seed=30)
    leaves = [t.detach().requires_grad_(True) for t in (x, res, w)]
    y, s = fa.layer_norm(leaves[0], leaves[2], residual=leaves[1])
    only = torch.autograd.grad(s, leaves[:2], gs, retain_graph=True)
    assert torch.equal(only[0], gs) and torch.equal(only[1], gs)
    got = torch.autograd.grad(y, leaves, gy)
    check_norm_grad((got[0], got[2]), norm_sum(x, res), norm_sum(x, res), w, None, gy, None, 1e-5,
                    torch.float32)
    y, s = fa.layer_norm(leaves[0], leaves[2], residual=leaves[0])
    twice, = torch.autograd.grad(y, leaves[0], gy)
    one = (2 * x).detach().requires_grad_(True)
    ref, = torch.autograd.grad(fa.layer_norm(one, w), one, gy)
    assert torch.equal(twice, 2 * ref)
    # accumulated into the leaves, in the same buffers
    a, c = (t.detach().clone().requires_grad_(True) for t in (x, res))
    for _ in range(2):
        y, s = fa.layer_norm(a, w, residual=c)
        torch.autograd.backward((y, s), (gy, gs))
    assert a.grad.data_ptr() != c.grad.data_ptr() and torch.equal(a.grad, c.grad)


def test_norm_keeps_what_it_says():
    x = rand(4096, 1024, seed=31, dtype=torch.bfloat16).requires_grad_(True)
    held = []
    for keep8 in (False, True):
        before = torch.cuda.memory_allocated()
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: (held.append(t.numel() * t.element_size()), t)[1], lambda t: t):
            y = fa.layer_norm(x, keep8=keep8)
        del y
        assert torch.cuda.memory_allocated() <= before
    assert sum(held) == 2 * x.numel() + 8 * 4096 + x.numel() * 17 // 16 + 8 * 4096
    y = fa.layer_norm(x * 1, keep8=True)
    y.sum().backward()
    base = (x.detach() * 1).requires_grad_(True)
    inner = base * 1
    y = fa.layer_norm(inner, keep8=False)
    inner.data.add_(0)  # not seen
    with torch.no_grad():
        inner.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# --------------------------------------------------------------------------- #
# activation
# --------------------------------------------------------------------------- #

def plain_gelu(x, approximate):
    return F.gelu(x, approximate=approximate)


def check_gelu(y, x, approximate, dtype):
    want = plain_gelu(x.double(), approximate)
    # Phi (or the tanh form's factor) to 8 2^-24 absolute
    within(y, want, U[dtype] * want.abs() * (1 + 2 * U[dtype]) + 8 * E * x.double().abs(), dtype)


def check_gelu_grad(dx, kept, gy, approximate, dtype):
    k = kept.double().requires_grad_(True)
    slope, = torch.autograd.grad(plain_gelu(k, approximate).sum(), k)
    want = slope * gy.double()
    within(dx, want, U[dtype] * want.abs() * (1 + 2 * U[dtype])
           + 16 * E * (1 + kept.double().abs()) * gy.double().abs(), dtype)


@pytest.mark.parametrize("approximate", ["none", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (3, 7), (2, 5, 64), (33, 1000), (40, 1001), (500, 256)])
def test_gelu(shape, dtype, approximate):
    x = (3 * rand(*shape, seed=40)).to(dtype)
    gy = rand(*shape, seed=41, dtype=dtype)
    leaf = x.clone().requires_grad_(True)
    y = fa.gelu8(leaf, approximate=approximate)
    assert y.shape == x.shape and y.dtype == dtype
    check_gelu(y.detach(), x, approximate, dtype)
    assert torch.equal(fa.gelu8(x, approximate=approximate), y.detach())
    dx, = torch.autograd.grad(y, leaf, gy)
    check_gelu_grad(dx, fa.unpack8(fa.pack8(x)), gy, approximate, dtype)


@pytest.mark.parametrize("approximate", ["none", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_over_its_range(dtype, approximate):
    x = torch.linspace(-14, 14, 28 * 512 + 1, device="cuda").to(dtype)
    x = torch.cat((x, torch.tensor([0.0, -0.0, 60.0, -60.0, 1e-5, -1e-5, 3e4, -3e4],
                                   device="cuda").to(dtype)))
    check_gelu(fa.gelu8(x, approximate=approximate), x, approximate, dtype)
    # each value a group of its own is kept exactly
    col = x[:, None].clone().requires_grad_(True)
    gy = torch.ones_like(col)
    dx, = torch.autograd.grad(fa.gelu8(col, approximate=approximate), col, gy)
    check_gelu_grad(dx, col.detach(), gy, approximate, dtype)


def test_gelu_of_what_is_not_finite():
    x = torch.tensor([math.inf, math.nan, 1.0], device="cuda")
    y = fa.gelu8(x)
    assert y[0] == math.inf and bool(y[1].isnan()) and bool(y[2].isfinite())


@pytest.mark.parametrize("view", [lambda t: t.mT, lambda t: t[:, 1:], lambda t: t[::2, 8:]])
def test_gelu_of_views_and_of_expanded_gradients(view):
    x = view(rand(136, 136, seed=42))
    leaf = x.detach().requires_grad_(True)
    y = fa.gelu8(leaf)
    check_gelu(y.detach(), x, "none", torch.float32)
    dx, = torch.autograd.grad(y.sum(), leaf)
    check_gelu_grad(dx, fa.unpack8(fa.pack8(x)), torch.ones_like(x), "none", torch.float32)
    gy = view(rand(136, 136, seed=43))
    dx, = torch.autograd.grad(fa.gelu8(leaf), leaf, gy)
    check_gelu_grad(dx, fa.unpack8(fa.pack8(x)), gy, "none", torch.float32)


# --------------------------------------------------------------------------- #
# products
# --------------------------------------------------------------------------- #

# rows, inputs, outputs, bias
LINEARS = [
    (1, 1, 1, True),
    (1, 64, 32, True),
    (2, 8, 8, False),
    (5, 7, 3, True),
    (17, 64, 64, True),
    (63, 65, 130, True),
    (64, 128, 128, False),
    (65, 136, 264, True),
    (200, 192, 768, False),
    (333, 517, 333, True),
    (1000, 256, 256, True),
    (1037, 1000, 72, True),
    (129, 40, 1030, True),
    (4000, 64, 128, True),
    (700, 520, 520, True),
    (20000, 16, 24, True),
    (3, 5000, 264, True),      # few tiles, a long sum
    (300, 64, 3000, True),
    (2500, 300, 20, False),
    (1030, 1100, 2056, True),
    (9990, 1304, 700, True),   # tall tiles: two waves of low ones
    (9990, 700, 1304, False),  # the same for dx
]


def linear_case(case, dtype, seed=0):
    t, k, m, bias = case
    x = (rand(t, k, seed=seed) * torch.exp(0.5 * rand(k, seed=seed + 1)) + 0.2).to(dtype)
    w = rand(m, k, seed=seed + 2, scale=k ** -0.5, dtype=dtype)
    b = rand(m, seed=seed + 3, dtype=dtype) if bias else None
    return x, w, b, rand(t, m, seed=seed + 4, dtype=dtype)


def check_product(got, a, b, bias, dtype):
    """got = a b^T + bias: float32 sums of k terms, rounded once."""
    a, b = a.double(), b.double()
    want = a @ b.mT
    tol = (8 + 4 * math.sqrt(a.shape[-1])) * E * (a.abs() @ b.abs().mT)
    if bias is not None:
        want, tol = want + bias.double(), tol + 2 * E * bias.double().abs()
    within(got, want, (1 + 2 * U[dtype]) * tol + U[dtype] * want.abs(), dtype)


def check_weight_grad(dw, db, x, gy, dtype):
    kept = fa.unpack8(fa.pack8(x)).double().reshape(-1, x.shape[-1])
    g = gy.double().reshape(-1, gy.shape[-1])
    t = g.shape[0]
    # roundings (or truncations, on the tensor cores) of a sum of t terms: each at
    # most 2^-23 of a partial sum, which is the sum of magnitudes at the very most
    # and its square root's share of it for signs that vary
    for got, want, size in ((dw, g.T @ kept, g.T.abs() @ kept.abs()),
                            (db, g.sum(0), g.abs().sum(0))):
        if got is not None:
            tol = U[dtype] * want.abs() + (8 + 4 * math.sqrt(t)) * E * size
            within(got, want, (1 + 2 * U[dtype]) * tol, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", LINEARS)
def test_linear(case, dtype):
    x, w, b, gy = linear_case(case, dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = fa.linear8(leaves[0], leaves[1], leaves[2] if b is not None else None)
    assert torch.equal(y.detach(), fa.linear8(x, w, b))
    check_product(y.detach(), x, w, b, dtype)
    got = torch.autograd.grad(y, leaves, gy)
    check_product(got[0], gy, w.mT, None, dtype)
    assert got[1].shape == w.shape and got[1].is_contiguous()
    check_weight_grad(got[1], got[2] if b is not None else None, x, gy, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_views(dtype):
    big = rand(2, 50, 300, seed=50, dtype=dtype)
    grad = rand(2, 50, 400, seed=51, dtype=dtype)
    w = rand(300, 160, seed=52, dtype=dtype)
    for x, gy, wt in ((big[..., 4:164], grad[..., 8:168], w[:160]),
                      (big[..., 1:161], grad[..., 3:163], w[:160]),
                      (big[:, ::2, :160], grad[:, ::2, :160], w[::2][:160 // 2]),
                      (big.transpose(0, 1)[..., :160], grad.transpose(0, 1)[..., :300], w),
                      (big[0, :, :160].mT.reshape(160, 50).mT, grad[0, :, :300], w)):
        m = min(wt.shape[0], gy.shape[-1])
        wt, gy = wt[:m], gy[..., :m]
        leaves = [x.detach().requires_grad_(True), wt.detach().requires_grad_(True)]
        y = fa.linear8(*leaves)
        check_product(y.detach(), x, wt, None, dtype)
        dx, dw = torch.autograd.grad(y, leaves, gy)
        check_product(dx, gy, wt.mT, None, dtype)
        check_weight_grad(dw, None, x, gy, dtype)


def test_linear_with_an_expanded_gradient_and_parts_that_need_none():
    x, w, b, _ = linear_case(LINEARS[8][:3] + (True,), torch.bfloat16)
    for need in ((True, False, False), (False, True, False), (False, False, True),
                 (True, True, False), (False, True, True)):
        leaves = [t.detach().clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        y = fa.linear8(*leaves)
        y.sum().backward()
        one = torch.ones_like(y)
        if need[0]:
            check_product(leaves[0].grad, one, w.mT, None, torch.bfloat16)
        check_weight_grad(leaves[1].grad, leaves[2].grad, x, one, torch.bfloat16)
        assert [t.grad is not None for t in leaves] == list(need)


def test_linear_keeps_what_it_says():
    x = rand(1024, 512, seed=53, dtype=torch.float16).requires_grad_(True)
    w = rand(128, 512, seed=54, dtype=torch.float16)
    for need, want in ((True, 1024 * 512 * 17 // 16), (False, 0)):
        sizes = []
        weight = w.clone().requires_grad_(need)
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: (sizes.append(t.numel() * t.element_size()), t)[1], lambda t: t):
            fa.linear8(x, weight)
        assert sum(sizes) == want + 128 * 512 * 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_under_autocast(dtype):
    x, w, b, gy = linear_case(LINEARS[10], torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    with torch.autocast("cuda", dtype=dtype):
        y = fa.linear8(*leaves)
    assert y.dtype == dtype
    check_product(y.detach(), x.to(dtype), w.to(dtype), b.to(dtype), dtype)
    got = torch.autograd.grad(y, leaves, gy.to(dtype))
    assert all(g.dtype == torch.float32 for g in got)
    check_weight_grad(got[1].to(dtype), got[2].to(dtype), x.to(dtype), gy.to(dtype), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_rows_that_are_not_finite_reach_their_own_columns_alone(dtype):
    x, w, _, gy = linear_case((100, 200, 64, False), dtype)
    x[7, 70], x[9, 199] = math.inf, math.nan
    leaf = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(fa.linear8(x, leaf), leaf, gy)
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[64:128], bad[192:] = True, True          # the groups of the two
    assert bool(dw[:, bad].isnan().all()) and bool(dw[:, ~bad].isfinite().all())


# --------------------------------------------------------------------------- #
# together
# --------------------------------------------------------------------------- #

def block(x, p):
    """Norm, product, activation, product, residual sum and norm."""
    y = fa.layer_norm(x, p[0], p[1], keep8=True)
    y = fa.linear8(fa.gelu8(fa.linear8(y, p[2], p[3])), p[4], p[5])
    return fa.layer_norm(y, p[6], p[7], residual=x, keep8=True)


def block_params(width, dtype, seed=60):
    return [1 + 0.1 * rand(width, seed=seed), 0.1 * rand(width, seed=seed + 1),
            rand(4 * width, width, seed=seed + 2, scale=width ** -0.5),
            0.1 * rand(4 * width, seed=seed + 3),
            rand(width, 4 * width, seed=seed + 4, scale=0.5 * width ** -0.5),
            0.1 * rand(width, seed=seed + 5),
            1 + 0.1 * rand(width, seed=seed + 6), 0.1 * rand(width, seed=seed + 7)]


class Kept64(torch.autograd.Function):
    """A float64 operator whose backward pass takes its input from the packed copy of
    `actual`, the float32 tensor that the operators themselves were given: packing a
    float32 rounding of the float64 input instead would move, by one step, the codes
    of the few values that lie within a rounding of the border between two."""

    @staticmethod
    def forward(ctx, fn, actual, x, *params):
        ctx.fn = fn
        ctx.save_for_backward(actual, x, *params)
        return fn(x, x, *params)

    @staticmethod
    def backward(ctx, g):
        actual, x, *params = ctx.saved_tensors
        kept = fa.unpack8(fa.pack8(actual)).double()
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_(True) for t in (kept, *params)]
            return (None, None, *torch.autograd.grad(ctx.fn(x, leaves[0], *leaves[1:]), leaves, g))


def norm64(x, kept, w, b):
    m = x.mean(-1, keepdim=True)
    r = 1 / ((x - m).square().mean(-1, keepdim=True) + 1e-5).sqrt()
    # value and weight slope at `kept`; the input's slope is the norm's formula there
    xh = (kept - m) * r

    class Slope(torch.autograd.Function):
        @staticmethod
        def forward(ctx, k, h):
            return h

        @staticmethod
        def backward(ctx, g):
            h = xh.detach()
            return r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True)), None
    return Slope.apply(kept, xh.detach()) * w + b


def linear64(x, k, w, b):
    return F.linear(k, w, b)


def block64(x, p, actual):
    """`actual`: the float32 inputs of the five operators."""
    y = Kept64.apply(norm64, actual[0], x, p[0], p[1])
    y = Kept64.apply(linear64, actual[1], y, p[2], p[3])
    y = Kept64.apply(lambda x, k: F.gelu(k), actual[2], y)
    y = Kept64.apply(linear64, actual[3], y, p[4], p[5])
    s = x + y
    return Kept64.apply(norm64, actual[4], s, p[6], p[7]), s


@torch.no_grad()
def block_inputs(x, p):
    y = [x, fa.layer_norm(x, p[0], p[1])]
    y.append(fa.linear8(y[1], p[2], p[3]))
    y.append(fa.gelu8(y[2]))
    y.append(x + fa.linear8(y[3], p[4], p[5]))
    return y


def test_a_block_of_them_against_float64():
    x = rand(300, 96, seed=61)
    p = block_params(96, torch.float32)
    gy, gs = rand(300, 96, seed=62), rand(300, 96, seed=63)
    leaves = [t.clone().requires_grad_(True) for t in (x, *p)]
    out = block(leaves[0], leaves[1:])
    got = torch.autograd.grad(out, leaves, (gy, gs))
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    ref = block64(wide[0], wide[1:], block_inputs(x, p))
    want = torch.autograd.grad(ref, wide, (gy.double(), gs.double()))
    for a, b in zip((*out, *got), (*ref, *want)):
        # five operators in a row, float32 sums of up to 400 terms of either sign each:
        # sqrt(400) 2^-24 = 1.2e-6 of a value's size an operator, and as much again for
        # its operands; below 1e-4 with room
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel < 1e-4, rel
    # and against the gradient without packing: 1/255 of the range of 64 values is at
    # most 2 % of their deviation, and averages
    plain = [t.detach().double().requires_grad_(True) for t in leaves]
    y = F.layer_norm(plain[0], (96,), plain[1], plain[2])
    y = F.linear(F.gelu(F.linear(y, plain[3], plain[4])), plain[5], plain[6])
    s = plain[0] + y
    exact = torch.autograd.grad((F.layer_norm(s, (96,), plain[7], plain[8]), s), plain,
                                (gy.double(), gs.double()))
    for a, b in zip(got, exact):
        assert float((a.double() - b).norm() / b.norm()) < 0.02


def train_step(x, p, gy, gs):
    leaves = [t.requires_grad_(True) for t in (x, *p)]
    out = block(leaves[0], leaves[1:])
    return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, (gy, gs)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_block_is_the_same_bits_every_time_and_on_another_stream(dtype):
    x, gy, gs = (rand(700, 192, seed=64 + i, dtype=dtype) for i in range(3))
    p = [t.to(dtype) for t in block_params(192, dtype)]
    want = train_step(x, p, gy, gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        with torch.cuda.stream(side):
            got = train_step(*[t.detach() if torch.is_tensor(t) else [u.detach() for u in t]
                               for t in (x, p, gy, gs)])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_of_blocks_replay_in_any_order():
    inputs = [[rand(257, 96, seed=70 + 5 * k + i, dtype=torch.bfloat16) for i in range(3)]
              for k in range(2)]
    p = [t.bfloat16() for t in block_params(96, torch.bfloat16)]

    def step(k):
        x, gy, gs = inputs[k]
        return train_step(x.detach(), [t.detach() for t in p], gy, gs)

    want = [step(k) for k in range(2)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(step(k))
    for k in (1, 0, 1):
        graphs[k].replay()
        torch.cuda.synchronize()
        step(1 - k)
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))
    for t in inputs[0]:
        t.mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[0], step(0)))


def test_second_derivatives_are_refused():
    x = rand(4, 64, seed=80).requires_grad_(True)
    w = rand(8, 64, seed=81).requires_grad_(True)
    for y in (fa.layer_norm(x), fa.layer_norm(x, keep8=True), fa.gelu8(x), fa.linear8(x, w)):
        with pytest.raises(RuntimeError, match="[Dd]ouble|once|second|create_graph"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 8)])
def test_no_rows(shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    n = shape[-1]
    w, b = (torch.ones(n, device="cuda", requires_grad=True) for _ in range(2))
    y, s = fa.layer_norm(x, w, b, residual=x)
    m = torch.ones(5, n, device="cuda", requires_grad=True)
    total = y.sum() + s.sum() + fa.gelu8(x).sum() + fa.linear8(x, m).sum()
    total.backward()
    assert x.grad.shape == shape and not any(bool(t.grad.any()) for t in (w, b, m))
    p = fa.pack8(x)
    assert fa.unpack8(p).shape == shape


def test_another_device_is_refused_and_the_current_one_is_kept():
    x = rand(4, 64, seed=82)
    with pytest.raises(TypeError):
        fa.layer_norm(x, torch.ones(64))
    with pytest.raises(TypeError):
        fa.linear8(x, torch.ones(4, 64))
    assert torch.cuda.current_device() == 0


# --------------------------------------------------------------------------- #
# calls that the rest does not make
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_weights_that_start_anywhere(dtype):
    x, _, _, _, gy, _ = norm_case(((33,), 1024, False, "both", False), dtype, seed=90)
    both = [(1 + 0.1 * rand(1030, seed=91 + i)).to(dtype)[i + 1:i + 1025] for i in range(2)]
    check_norm(fa.layer_norm(x, *both), x, *both, 1e-5, dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, *both)]
    got = torch.autograd.grad(fa.layer_norm(*leaves, keep8=True), leaves, gy)
    check_norm_grad(got, x, fa.unpack8(fa.pack8(x)), *both, gy, None, 1e-5, dtype)


def test_vectors_are_rows():
    x = rand(200, seed=92).requires_grad_(True)
    w = rand(5, 200, seed=93).requires_grad_(True)
    for dtype in (torch.float32, torch.bfloat16):
        a, m = (t.detach().to(dtype).requires_grad_(True) for t in (x, w))
        for fn, leaves in ((lambda t: fa.layer_norm(t, keep8=True), (a,)), (fa.gelu8, (a,)),
                           (lambda t: fa.linear8(t, m), (a, m))):
            y = fn(a)
            two = fn(a[None])
            assert y.dim() == 1 and torch.equal(y, two[0])
            g = rand(*y.shape, seed=94, dtype=dtype)
            for p, q in zip(torch.autograd.grad(y, leaves, g),
                            torch.autograd.grad(two, leaves, g[None])):
                assert torch.equal(p, q)


@pytest.mark.parametrize("scale", [2.0 ** -24, 2.0 ** -20, 2.0 ** -17])
def test_linear_of_float16_spreads_whose_steps_float16_does_not_hold(scale):
    x = (rand(70, 200, seed=95) * scale * 8).half()
    x[3] = 0.5                                    # and rows that it does hold
    x[5, :64] += rand(64, seed=96).half()
    w, gy = rand(24, 200, seed=97, dtype=torch.float16), rand(70, 24, seed=98, dtype=torch.float16)
    w.requires_grad_(True)
    dw, = torch.autograd.grad(fa.linear8(x, w), w, gy)
    check_weight_grad(dw, None, x, gy, torch.float16)


def test_kept_values_that_are_moved_to_the_host_and_back():
    x = rand(130, 192, seed=100, dtype=torch.bfloat16)
    p = [t.bfloat16() for t in block_params(192, torch.bfloat16)]
    gy, gs = (rand(130, 192, seed=101 + i, dtype=torch.bfloat16) for i in range(2))
    want = train_step(x.clone(), [t.clone() for t in p], gy, gs)
    with torch.autograd.graph.save_on_cpu():
        got = train_step(x.clone(), [t.clone() for t in p], gy, gs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_products_on_two_streams_at_once():
    cases = [linear_case((2000, 512, 768, True), torch.bfloat16, seed=110 + 7 * i) for i in range(2)]

    def step(x, w, b, gy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = fa.linear8(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(step(*c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_the_first_calls_of_a_process_may_be_captured():
    import textwrap
    from conftest import REPO
    code = textwrap.dedent(f"""
        import sys, torch
        sys.path.insert(0, {str(REPO)!r})
        import frame_analytics_b200 as fa
        g = torch.Generator(device="cuda").manual_seed(0)
        x, gy = (torch.randn(300, 192, generator=g, device="cuda").bfloat16() for _ in range(2))
        w = torch.randn(192, 192, generator=g, device="cuda").bfloat16()
        def step():
            a, m = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            y = fa.gelu8(fa.linear8(fa.layer_norm(a, keep8=True), m))
            return (y.detach(), *torch.autograd.grad(y, (a, m), gy))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        print("same")
    """)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr


def test_the_example_runs_with_kept_activations_and_its_gradients_are_close():
    from conftest import REPO
    sys.path.insert(0, str(REPO / "examples"))
    import train_restoration

    losses = train_restoration.train(steps=3, size=64, frames=2, keep8=True)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
    g = torch.Generator(device="cuda").manual_seed(1)
    clean, noisy = train_restoration.batch(2, 64, g, "cuda")
    grads = []
    for keep8 in (False, True):
        torch.manual_seed(0)
        net = train_restoration.Restorer(keep8=keep8).cuda()
        torch.nn.init.normal_(net.head.weight, std=0.02)
        loss = fa.mse(clean.double(), net(noisy).double())
        loss.backward()
        grads.append([p.grad for p in net.parameters()])
    for a, b in zip(*grads):
        # each kept value is off by at most 1/255 of the range of 64: under 2 % of its
        # deviation, and the same operators exactly otherwise
        assert float((a.double() - b.double()).norm()) <= 0.05 * float(b.double().norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sums_of_many_terms_of_one_sign(dtype):
    """Longer than one chunk of a tensor-core sum, whose additions truncate."""
    x = rand(1_100_000, 16, seed=120).abs().to(dtype)
    gy = (2.0 ** -10 * rand(1_100_000, 24, seed=121).abs()).to(dtype)
    w = rand(24, 16, seed=122, dtype=dtype).requires_grad_(True)
    b = rand(24, seed=123, dtype=dtype).requires_grad_(True)
    dw, db = torch.autograd.grad(fa.linear8(x, w, b), (w, b), gy)
    kept = fa.unpack8(fa.pack8(x)).double()
    for got, want in ((dw, gy.double().T @ kept), (db, gy.double().sum(0))):
        # chunks of 32768 terms: 2048 additions, each at most 2^-24 of the sum short;
        # column sums: a few thousand rounded additions
        tol = (U[dtype] + 2048 * E) * want.abs()
        within(got, want, (1 + 2 * U[dtype]) * tol, dtype)


def test_products_over_more_inputs_than_a_chunk():
    x = rand(5000, 33000, seed=124, dtype=torch.bfloat16)
    w = rand(1000, 33000, seed=125, dtype=torch.bfloat16)
    y = fa.linear8(x, w)
    check_product(y[::7], x[::7], w, None, torch.bfloat16)
    leaf = x[:200].clone().requires_grad_(True)
    gy = rand(200, 1000, seed=126, dtype=torch.bfloat16)
    dx, = torch.autograd.grad(fa.linear8(leaf, w), leaf, gy)
    check_product(dx, gy, w.mT, None, torch.bfloat16)


def test_wide_rows_take_a_workspace_of_their_own_size():
    """Parts of the column sums as there are rows for, not as there are multiprocessors."""
    x = rand(3, 1 << 22, seed=130, dtype=torch.bfloat16).requires_grad_(True)
    w = rand(1 << 22, seed=131).requires_grad_(True)
    y = fa.layer_norm(x, w)
    gy = torch.ones_like(y)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    _, dw = torch.autograd.grad(y, (x, w), gy)
    assert torch.cuda.max_memory_allocated() - before <= 8 * x.numel() * x.element_size()
    mean, var = x.detach().double().mean(1, True), x.detach().double().var(1, False, keepdim=True)
    want = ((x.detach().double() - mean) / (var + 1e-5).sqrt()).sum(0)
    # mean and variance of 2^22 float32 terms, 2^14 in a lane's row: 2^14 steps each, of
    # which the values, below 8, take all, and then three additions of them
    assert float((dw.double() - want).abs().max()) <= 3 * 8 * 2.0 ** 14 * E + 8 * 4 * E

    inputs = rand(3, 8, seed=132, dtype=torch.bfloat16)
    weight = rand(1 << 21, 8, seed=133, dtype=torch.bfloat16)
    bias = torch.zeros(1 << 21, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = fa.linear8(inputs, weight, bias)
    gy = torch.ones_like(y)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    db, = torch.autograd.grad(y, bias, gy)
    assert torch.cuda.max_memory_allocated() - before <= 8 * y.numel() * y.element_size()
    assert torch.equal(db, torch.full_like(db, 3.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,pitch", [(939, 960), (57, 64), (1, 64), (65, 128), (63, 64), (8, 64),
                                         (200, 256), (939, 968), (57, 60)])
def test_rows_padded_to_a_pitch(width, pitch, dtype):
    """Rows at a pitch of whole groups: neighbouring lanes' places then lie 8 values apart
    across the gaps, too."""
    x = rand(41, pitch, seed=140, dtype=dtype)[:, :width]
    g = rand(41, pitch, seed=141, dtype=dtype)[:, :width]
    got, want = fa.pack8(x), fa.pack8(x.contiguous())
    assert torch.equal(got.codes, want.codes) and torch.equal(got.ranges, want.ranges)
    assert torch.equal(fa.gelu8(x), fa.gelu8(x.contiguous()))
    w = rand(24, width, seed=142, dtype=dtype)
    results = []
    for a, b in ((x, g), (x.contiguous(), g.contiguous())):
        leaf, wl = a.detach().requires_grad_(True), w.clone().requires_grad_(True)
        dx, = torch.autograd.grad(fa.gelu8(leaf), leaf, b)
        dn, = torch.autograd.grad(fa.layer_norm(leaf, keep8=True), leaf, b)
        dw, = torch.autograd.grad(fa.linear8(leaf, wl), wl, b[:, :1].expand(41, 24))
        results.append((dx, dn, dw))
    assert all(torch.equal(p, q) for p, q in zip(*results))


@pytest.mark.parametrize("rows,inputs,outputs", [(510, 1024, 4096), (9001, 200, 264), (4080, 256, 1000)])
def test_a_bias_gradient_beside_the_weights_is_the_same_bits(rows, inputs, outputs):
    """The two run at the same time where there is room; alone, and in a graph, they do not."""
    x, g = (rand(rows, n, seed=150, dtype=torch.bfloat16) for n in (inputs, outputs))
    w = rand(outputs, inputs, seed=151, dtype=torch.bfloat16).requires_grad_(True)
    b = rand(outputs, seed=152, dtype=torch.bfloat16).requires_grad_(True)
    alone = [torch.autograd.grad(fa.linear8(x, w, b), t, g)[0] for t in (w, b)]
    for _ in range(10):
        dw, db = torch.autograd.grad(fa.linear8(x, w, b), (w, b), g)
        # the results' memory is free for others when the call returns
        y = fa.linear8(x, w.detach(), b.detach())
        assert torch.equal(dw, alone[0]) and torch.equal(db, alone[1])
        del dw, db, y
    # the sum of at most 9001 rows is off by t (a row's additions pass through no more than
    # 4096 roundings), and its rounding to the dtype by U of what it then is: U (|sum| + t)
    want, t = g.double().sum(0), 4096 * E * g.double().abs().sum(0)
    within(alone[1], want, t + U[torch.bfloat16] * (want.abs() + t), torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dw, db = torch.autograd.grad(fa.linear8(x, w, b), (w, b), g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dw, alone[0]) and torch.equal(db, alone[1])


def test_float32_sums_of_many_terms_of_one_sign():
    """More tiles than run at once: the rows' parts are there for the sum's sake alone."""
    rows = 200_001
    x = (1.0 + rand(rows, 1, seed=160).abs()).expand(rows, 2560).contiguous()
    g = (1.0 + rand(rows, 1, seed=161).abs()).expand(rows, 2048).contiguous()
    w = rand(2048, 2560, seed=162).requires_grad_(True)
    dw, = torch.autograd.grad(fa.linear8(x, w), w, g)
    kept = fa.unpack8(fa.pack8(x[:, :1].contiguous())).double()
    want = (g[:, :1].double() * kept).sum()
    # parts of at most 32768 terms, each addition off by E of the part's sum at most: on
    # average half of it, as the sum grows evenly; 7 additions of parts, one a product's
    tol = (0.51 * 32768 + 32 + 7) * E * float(want)
    assert float((dw.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("what", ["value", "gradient"])
def test_a_thread_may_make_its_first_call_here(what):
    """A thread that has launched nothing has no context of its own yet."""
    import textwrap
    from conftest import REPO
    code = textwrap.dedent(f"""
        import sys, threading, torch
        sys.path.insert(0, {str(REPO)!r})
        import frame_analytics_b200 as fa
        x, gy = (torch.randn(256, 128, device="cuda").bfloat16() for _ in range(2))
        w = torch.randn(128, 128, device="cuda").bfloat16().requires_grad_({what == "gradient"})
        q = fa.orthogonalize(x)
        got = []
        if {what == "gradient"}:             # autograd's own thread
            grad, = torch.autograd.grad(fa.linear8(x, w), w, gy)
            got.append(torch.equal(grad, torch.autograd.grad(fa.linear8(x, w), w, gy)[0]))
        else:
            y = fa.linear8(x, w)
            spare = [torch.empty_like(y) for _ in range(4)]
            del spare                        # the allocator has what the threads take
            calls = ((lambda: fa.linear8(x, w), y), (lambda: fa.orthogonalize(x), q))
            def run(call, want):
                a = call()
                got.append(torch.equal(a, want))
            for call in calls:
                t = threading.Thread(target=run, args=call)
                t.start()
                t.join()
        assert len(got) == (1 if {what == "gradient"} else 2) and all(got), got
        print("same")
    """)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,inputs,outputs", [(200, 256, 256), (1600, 512, 256), (700, 1100, 520)])
def test_a_weight_gradient_sees_every_stage_as_written(rows, inputs, outputs, dtype):
    """Both blocks of a pair write the stages that one of them multiplies.  Calls on other
    values in between, so that a stage read too early would hold something else."""
    cases = [linear_case((rows, inputs, outputs, False), dtype, seed=170 + 7 * i) for i in range(2)]
    leaves = [w.detach().requires_grad_(True) for _, w, _, _ in cases]

    def grad(i):
        return torch.autograd.grad(fa.linear8(cases[i][0], leaves[i]), leaves[i], cases[i][3])[0]

    want = [grad(i) for i in range(2)]
    for dw, (x, _, _, gy) in zip(want, cases):
        check_weight_grad(dw, None, x, gy, dtype)
    for k in range(60):
        assert torch.equal(grad(k % 2), want[k % 2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 24, 192, 577, 1024, 4096, 8192, 20480, 32760, 40000])
def test_norm_of_rows_of_one_value_is_nothing(width, dtype):
    """Whatever the value: its mean is itself, which a plain float32 sum misses."""
    values = torch.cat((torch.tensor([0.37, 1234.567, -998.2, 3.3e4], device="cuda"),
                        1000 + 30 * rand(36, seed=180)))[:, None].to(dtype)
    x = values.expand(40, width).contiguous()
    w, b = 1 + rand(width, seed=181).abs(), rand(width, seed=182)
    for keep8 in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = fa.layer_norm(*leaves, keep8=keep8)
        assert torch.equal(y.detach(), b.to(dtype).expand(40, width))
        gy = torch.ones_like(y)
        dw, db = torch.autograd.grad(y, leaves[1:], gy)
        # each distance is nothing, and 40 is a float32 number
        assert not bool(dw.any()) and bool((db == 40).all())


@pytest.mark.parametrize("width", [192, 577, 1024, 4096, 40000])
def test_norm_of_a_row_whose_spread_is_small_against_its_offset(width):
    x = 1000 + 0.01 * rand(64, width, seed=183)
    m = x.double().mean(1, keepdim=True)
    r = 1 / ((x.double() - m).square().mean(1, keepdim=True) + 1e-5).sqrt()
    want = (x.double() - m) * r
    # The mean that is taken off is rounded to float32 once, E |m|, behind a first one m0
    # that is at most e0 = (n / 32 + 80) E |m| off and a mean of distances from m0, which
    # is as far off relative to them (|d| <= |s - m| + e0); the mean of d^2, the variance
    # and at most e0^2, likewise, and half of that is 1 / deviation's.
    rel = (width / 32 + 80) * E
    e0 = rel * m.abs()
    em = E * m.abs() + rel * ((x.double() - m).abs().mean(1, keepdim=True) + e0)
    tol = (em + 2 * E * (x.double() - m).abs()) * r + want.abs() * (rel * (1 + 2 * (e0 * r) ** 2) + 8 * E)
    within(fa.layer_norm(x), want, tol + E * want.abs(), torch.float32)


@pytest.mark.parametrize("approximate", ["none", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_far_out_relative_to_its_value(dtype, approximate):
    """Down to -13, where values and slopes are 1e-37 (tanh form: nothing).

    Both are at most (32 + 2 x^2) E of their terms off: 20 E of the tail's factor (1.1e-6)
    and its rounding, 4 E of an approximate exponential, the roundings of an exponent of
    x^2 / 2 (three, of a value that the exponential takes absolutely) and of the few
    operations around; the tanh form with its own exponent 2 u, four roundings, in place of
    x^2 / 2.  float32's library functions are closer than that."""
    x = torch.linspace(-13, 13, 26 * 512 + 1, device="cuda").to(dtype)[:, None]
    leaf = x.clone().requires_grad_(True)       # each value a group of its own: kept exactly
    y = fa.gelu8(leaf, approximate=approximate)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(x))
    d = x.double()
    if approximate == "tanh":
        c = (2 / math.pi) ** 0.5
        two_u, up = 2 * c * (d + 0.044715 * d ** 3), 2 * c * (1 + 3 * 0.044715 * d * d)
        f = torch.sigmoid(two_u)
        value, first, second = d * f, f, d * f * torch.sigmoid(-two_u) * up
        rel = (32 + 4 * two_u.abs()) * E
        # above zero f (1 - f) is within E, a rounding of f
        extra = torch.where(d > 0, 2 * E * d * up, 0.0)
    else:
        first = torch.special.erfc(-d / 2 ** 0.5) / 2
        value, second = d * first, d * torch.exp(-d * d / 2) / (2 * math.pi) ** 0.5
        rel, extra, up = (32 + 2 * d * d) * E, torch.zeros_like(d), d.abs()
    # A factor f (or an exponential) below 2^-126 may be flushed, which moves f by that,
    # the value x f by |x| of it, and the slope f + x f (1 - f) up by 1 + |x| up of it
    # (the other form's x exp(-x^2 / 2): by |x|)
    low = 2.0 ** -126
    for got, want, size, by in ((y.detach(), value, value.abs(), 1 + d.abs()),
                                (dx, first + second, first + second.abs(), 1 + d.abs() * (1 + up))):
        tol = rel * size + (0 if got is not dx else extra) + low * by
        within(got, want, U[dtype] * want.abs() + (1 + 2 * U[dtype]) * tol, dtype)


@pytest.mark.parametrize("dtype,rows,inputs,outputs", [
    (torch.bfloat16, 131_073, 2304, 2304),     # more tiles than pairs of blocks, five chunks
    (torch.float16, 100_000, 2304, 2304),
    (torch.bfloat16, 300_001, 520, 260),       # fewer, cut into parts of a few chunks each
    (torch.bfloat16, 1_000_003, 1024, 1024),
    (torch.float32, 70_001, 2304, 2304),
    (torch.float32, 150_001, 520, 260),
])
def test_weight_gradients_of_many_rows_take_little_memory(dtype, rows, inputs, outputs):
    """Sums of many chunks, in a workspace that does not depend on how many."""
    # each row is one of 64, so that what the sums come to is known in float64 at once
    bx, bg = (rand(64, n, seed=190 + i, dtype=dtype) for i, n in enumerate((inputs, outputs)))
    at = torch.arange(rows, device="cuda") % 64
    at[: rows // 3] = at[: rows // 3].flip(0)
    x, g = bx[at], bg[(at * 7 + 3) % 64]
    w = rand(outputs, inputs, seed=192, dtype=dtype).requires_grad_(True)
    y = fa.linear8(x, w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dw, = torch.autograd.grad(y, w, g)
    scratch = torch.cuda.max_memory_allocated() - before - dw.numel() * dw.element_size()
    # eight slabs a pair of blocks, and a copy of rows that are not whole 16 bytes
    copy = rows * 264 * 2 if outputs == 260 and dtype != torch.float32 else 0
    assert scratch <= 8 * 74 * 2 ** 18 + copy + (1 << 20), scratch
    many = torch.bincount(at, minlength=64).double()[:, None]
    kept = fa.unpack8(fa.pack8(bx)).double()
    bg = bg[(torch.arange(64, device="cuda") * 7 + 3) % 64].double()
    want, size = bg.T @ (kept * many), bg.T.abs() @ (kept.abs() * many)
    # The rows repeat, so roundings repeat too and add up: of a sum of 32768 terms every
    # addition (16 terms each on the tensor cores, which truncate: a whole step) may be off by
    # E (2 E) of what the sum then is, at most `size`; then a rounding a chunk or a part.
    steps = 32768 if dtype == torch.float32 else 2 * 2048
    tol = U[dtype] * want.abs() + (steps + 32 + rows / 32768) * E * size
    past = want.abs() > torch.finfo(dtype).max * (1 - 2 * U[dtype])   # rounded to infinity
    within(dw[~past], want[~past], ((1 + 2 * U[dtype]) * tol)[~past], dtype)
    assert bool((dw[past].sign() == want[past].sign()).all())
    assert torch.equal(dw, torch.autograd.grad(fa.linear8(x, w), w, g)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_of_many_tiles_over_more_inputs_than_a_chunk(dtype):
    rows, inputs, outputs = 5200, 40_000, 1100
    x, w = rand(rows, inputs, seed=195, dtype=dtype), rand(outputs, inputs, seed=196, dtype=dtype)
    b = rand(outputs, seed=197, dtype=dtype)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = fa.linear8(x, w, b)
    scratch = torch.cuda.max_memory_allocated() - before - y.numel() * y.element_size()
    # a slab a pair of blocks; float32: three parts of the result
    most = 74 * 2 ** 18 if dtype != torch.float32 else 12 * rows * outputs
    assert scratch <= most + (1 << 20), scratch
    check_product(y[::13], x[::13], w, b, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_block_under_autocast(dtype):
    """A float32 residual stream and weights around products in 16 bits."""
    x, gy = rand(300, 96, seed=200), rand(300, 96, seed=201)
    p = block_params(96, torch.float32, seed=202)
    leaves = [t.clone().requires_grad_(True) for t in (x, *p)]
    with torch.autocast("cuda", dtype=dtype):
        y, s = block(leaves[0], leaves[1:])
    assert y.dtype == s.dtype == torch.float32
    got = torch.autograd.grad((y, s), leaves, (gy, gy))
    assert all(g.dtype == torch.float32 and g.shape == t.shape for g, t in zip(got, leaves))
    # the same with every change of type written out
    again = [t.clone().requires_grad_(True) for t in (x, *p)]
    q = again[1:]
    h = fa.layer_norm(again[0], q[0], q[1], keep8=True).to(dtype)
    h = fa.gelu8(fa.linear8(h, q[2].to(dtype), q[3].to(dtype)))
    h = fa.linear8(h, q[4].to(dtype), q[5].to(dtype)).float()
    want = fa.layer_norm(h, q[6], q[7], residual=again[0], keep8=True)
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    for a, b in zip(got, torch.autograd.grad(want, again, (gy, gy))):
        assert torch.equal(a, b)


def test_norm_operands_of_two_types_meet_in_float32_under_autocast():
    x, w, b = rand(9, 64, seed=203), 1 + rand(64, seed=204).abs(), rand(64, seed=205)
    half, bf = torch.float16, torch.bfloat16
    with torch.autocast("cuda", dtype=bf):
        for a, r in ((bf, torch.float32), (torch.float32, half), (half, bf)):
            y, s = fa.layer_norm(x.to(a), w, b, residual=x.to(r))
            want, t = fa.layer_norm(x.to(a).float(), w, b, residual=x.to(r).float())
            assert torch.equal(y, want) and torch.equal(s, t) and y.dtype == torch.float32
        # what fits is left as it is
        y, s = fa.layer_norm(x.to(bf), w, b, residual=x.to(bf))
        assert y.dtype == s.dtype == bf
        assert fa.layer_norm(x.to(bf), w.to(bf), b.to(bf)).dtype == bf
        for wt, bt in ((half, half), (half, torch.float32), (bf, torch.float32), (half, None)):
            bias = None if bt is None else b.to(bt)
            y = fa.layer_norm(x.to(bf), w.to(wt), bias)
            want = fa.layer_norm(x.to(bf), w.to(wt).float(), None if bias is None else bias.float())
            assert torch.equal(y, want) and y.dtype == bf
        with pytest.raises(ValueError, match="residual"):
            fa.layer_norm(x, residual=x[:3].half())
        with pytest.raises(TypeError, match="weight"):
            fa.layer_norm(x, w.double())
    with pytest.raises(ValueError, match="residual"):
        fa.layer_norm(x, residual=x.half())


def test_a_wait_that_gives_up_is_reported_by_the_next_call():
    """A product's own waits, which sleep: a phase that nothing completes, with nothing in
    flight, for 50 ms.  A second wait behind it gives up without its own 50 ms."""
    from frame_analytics_b200 import _cabi
    L = _cabi.load()
    x, w, b, _ = linear_case((300, 200, 264, True), torch.bfloat16, seed=210)
    want = fa.linear8(x, w, b)
    t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    stream = torch.cuda.current_stream().cuda_stream
    t[0].record()
    assert L.fa_b200_linear8_wait_selftest(50_000_000, 0, stream) == 0
    t[1].record()
    torch.cuda.synchronize()
    # the clock is looked at behind every sixteenth poll, of 2 ms at most, and so is the
    # word that says that a wait has given up: 50 and twice 16 x 2, and not twice 50 and that
    assert 50 <= t[0].elapsed_time(t[1]) < 50 + 2 * 32 + 10
    with pytest.raises(_cabi.KernelError, match="timed out"):
        fa.linear8(x, w, b)
    assert torch.equal(fa.linear8(x, w, b), want)


@pytest.mark.parametrize("shape", [(9, 1), (2, 5, 1), (1,), (9, 66)])
def test_imaginary_parts_keep_their_sign(shape):
    """The imaginary part of a conjugate, and the gradient of one, are views whose sign is
    not in memory; a column of them needs no copy for its strides."""
    def imag(seed, *shape):
        c = torch.complex(rand(*shape, seed=seed), rand(*shape, seed=seed + 1))
        view = c.conj().imag
        assert view.is_neg()
        return view, -c.imag.contiguous()

    n = shape[-1]
    pairs = [imag(220 + 2 * i, *s) for i, s in enumerate((shape, shape, (n,), (n,), (3, n), (3,)))]
    p, q = fa.pack8(pairs[0][0]), fa.pack8(pairs[0][1])
    assert torch.equal(p.codes, q.codes) and torch.equal(p.ranges, q.ranges)
    results = []
    for k in range(2):
        x, r, w, b, m, c = (pair[k].detach().requires_grad_(True) for pair in pairs)
        gy = pairs[1][k]
        y, s = fa.layer_norm(x, w, b, residual=r, keep8=True)
        a = fa.gelu8(x)
        z = fa.linear8(x, m, c)
        column = fa.linear8(x, m[:1], c[:1])
        results.append([t.detach() for t in (y, s, a, z, column)])
        results[-1] += torch.autograd.grad((y, s), (x, r, w, b), (gy, gy))
        results[-1] += torch.autograd.grad(a, x, gy)
        results[-1] += torch.autograd.grad(z, (x, m, c), torch.ones_like(z))
        results[-1] += torch.autograd.grad(column, (x, m, c), gy[..., :1])
        with torch.no_grad():
            results[-1] += [fa.layer_norm(x, w, b), fa.linear8(x, m, c)]
    for got, want in zip(*results):
        assert torch.equal(got, want)


@pytest.mark.parametrize("width", [2112, 2111])
def test_norm_and_gelu_past_2_31_values(width):
    """Rows stand alone, so those at either end are the bits of a call on them."""
    rows = (1 << 31) // width + 77
    x = torch.full((rows, width), 0.5, dtype=torch.bfloat16, device="cuda")
    g = torch.full((rows, width), 0.25, dtype=torch.bfloat16, device="cuda")
    ends = [slice(0, 40), slice(rows - 40, rows)]
    for i, part in enumerate(ends):
        x[part], g[part] = (rand(40, width, seed=230 + 2 * i + k).bfloat16() for k in range(2))
    w = (1 + 0.1 * rand(width, seed=235)).bfloat16()
    for call in (lambda t: fa.layer_norm(t, w, residual=t, keep8=True)[0],
                 lambda t: fa.layer_norm(t, w), fa.gelu8):
        leaf = x.detach().requires_grad_(True)
        y = call(leaf)
        dx, = torch.autograd.grad(y, leaf, g)
        for part in ends:
            small = x[part].clone().requires_grad_(True)
            want = call(small)
            assert torch.equal(y[part], want)
            assert torch.equal(dx[part], torch.autograd.grad(want, small, g[part])[0])
        del y, dx


@pytest.mark.parametrize("dtype,inputs", [(torch.bfloat16, 2112), (torch.bfloat16, 2111),
                                          (torch.float32, 2111)])
def test_products_past_2_31_values(dtype, inputs):
    """Inputs and results of more than 2^31 values, in rows that are all nothing but at
    their ends: the weight's gradient is that of the ends."""
    rows, outputs = (1 << 31) // 2111 + 77, 2112
    x = torch.zeros(rows, inputs, dtype=dtype, device="cuda")
    g = torch.zeros(rows, outputs, dtype=dtype, device="cuda")
    ends = [slice(0, 40), slice(rows - 40, rows)]
    for i, part in enumerate(ends):
        x[part], g[part] = (rand(40, n, seed=240 + 2 * i + k).to(dtype)
                            for k, n in enumerate((inputs, outputs)))
    w = rand(outputs, inputs, seed=245, scale=inputs ** -0.5).to(dtype).requires_grad_(True)
    leaf = x.detach().requires_grad_(True)
    y = fa.linear8(leaf, w)
    dx, dw = torch.autograd.grad(y, (leaf, w), g)
    for part in ends:
        check_product(y[part].detach(), x[part], w.detach(), None, dtype)
        check_product(dx[part], g[part], w.detach().mT, None, dtype)
    assert not bool(y[40:80].any()) and not bool(dx[rows - 80:rows - 40].any())
    both = [torch.cat([t[part] for part in ends]) for t in (x, g)]
    check_weight_grad(dw, None, *both, dtype)


def test_float32_tanh_slopes_are_as_close_as_their_terms():
    """f + x f (1 - f) 2 u' with f = 1 / (1 + e), e = exp(-2 u): e is off by 4 E of itself
    (2 ulp) and the exponent's roundings, five of 2 u at most; f by two roundings and what
    e's error moves it, f (1 - f) of that; the second term by as much twice and a dozen
    roundings of its own.  A rounding of f itself, where f is near one and 1 - f is small,
    is nothing to the second term."""
    x = torch.linspace(-6, 13, 19 * 512 + 1, device="cuda")[:, None]
    leaf = x.clone().requires_grad_(True)       # each value a group of its own: kept exactly
    dx, = torch.autograd.grad(fa.gelu8(leaf, approximate="tanh"), leaf, torch.ones_like(x))
    d = x.double()
    c = (2 / math.pi) ** 0.5
    two_u, up = 2 * c * (d + 0.044715 * d ** 3), 2 * c * (1 + 3 * 0.044715 * d * d)
    f, rest = torch.sigmoid(two_u), torch.sigmoid(-two_u)
    second = d * f * rest * up
    of_e = (4 + 5 * two_u.abs()) * E
    tol = 2 * E * f + f * rest * of_e + second.abs() * (2 * of_e + 12 * E)
    within(dx, f + second, 1.01 * tol + E * (f + second).abs(), torch.float32)
