"""The 8-bit block operators' refusals, which need no GPU."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

import frame_analytics_b200 as fa
from frame_analytics_b200 import _cabi, block


@pytest.mark.parametrize("call", [fa.pack8, fa.gelu8, fa.layer_norm],
                         ids=["pack8", "gelu8", "layer_norm"])
@pytest.mark.parametrize("x,exc", [
    (torch.zeros(2, 3), TypeError),                              # not on the GPU
    (torch.zeros(2, 3, dtype=torch.float64), TypeError),
    (torch.zeros(2, 3, dtype=torch.int32), TypeError),
    (torch.tensor(1.0), ValueError),
    (torch.zeros(2, 0), ValueError),
    ([1.0, 2.0], TypeError),
])
def test_values_are_refused(call, x, exc):
    with pytest.raises(exc):
        call(x)


def test_rows_past_the_limits_are_refused():
    one = torch.zeros(1)
    with pytest.raises(ValueError, match="last dimension"):
        fa.layer_norm(one.expand(2, (1 << 24) + 1))
    with pytest.raises(ValueError, match="last dimension"):
        fa.pack8(one.expand(1 << 31))
    with pytest.raises(ValueError, match="last dimension"):
        fa.linear8(one.expand(2, 1 << 22), one.expand(3, 1 << 22))
    for x, w in ((one.expand(2, 4), one.expand(1 << 22, 4)),
                 (one.expand((1 << 27) + 1, 4), one.expand(2, 4))):
        with pytest.raises(ValueError, match="rows"):
            fa.linear8(x, w)


@pytest.mark.parametrize("kw,exc", [
    ({}, TypeError),                                             # not on the GPU
    ({"weight": torch.ones(7)}, ValueError),
    ({"weight": torch.ones(1, 8)}, ValueError),
    ({"weight": torch.ones(8, dtype=torch.float64)}, TypeError),
    ({"x": torch.zeros(3, 8).half(), "weight": torch.ones(8, dtype=torch.bfloat16)}, TypeError),
    ({"x": torch.zeros(3, 8).half(), "weight": torch.ones(8), "bias": torch.ones(8).half()},
     ValueError),
    ({"bias": torch.ones(9)}, ValueError),
    ({"bias": [0.0] * 8}, TypeError),
    ({"residual": 1.0}, TypeError),
    ({"residual": torch.zeros(8)}, ValueError),                  # no broadcast
    ({"residual": torch.zeros(3, 8).half()}, ValueError),
    ({"eps": -1e-5}, ValueError),
    ({"eps": float("nan")}, ValueError),
    ({"eps": float("inf")}, ValueError),
])
def test_layer_norm_refuses(kw, exc):
    args = dict(x=torch.zeros(3, 8))
    args.update(kw)
    with pytest.raises(exc):
        fa.layer_norm(**args)


def test_gelu8_refuses_other_forms():
    with pytest.raises(ValueError, match="approximate"):
        fa.gelu8(torch.zeros(4), approximate="quick")


@pytest.mark.parametrize("kw,exc", [
    ({}, TypeError),                                             # not on the GPU
    ({"x": torch.zeros(3, 7)}, ValueError),
    ({"x": torch.zeros(3, 8).half()}, ValueError),
    ({"x": torch.zeros(3, 8, dtype=torch.float64)}, TypeError),
    ({"weight": torch.zeros(8)}, ValueError),
    ({"weight": torch.zeros(0, 8)}, ValueError),
    ({"weight": None}, ValueError),
    ({"bias": torch.zeros(4)}, ValueError),
    ({"bias": 0.0}, TypeError),
    ({"bias": torch.zeros(5).half()}, ValueError),
])
def test_linear8_refuses(kw, exc):
    args = dict(x=torch.zeros(3, 8), weight=torch.zeros(5, 8))
    args.update(kw)
    with pytest.raises(exc):
        fa.linear8(**args)


def packed(**kw):
    p = fa.Packed8(torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.int32),
                   torch.Size((3, 100)), torch.bfloat16)
    return p._replace(**kw)


@pytest.mark.parametrize("p,exc", [
    (packed(), TypeError),                                       # not on the GPU
    (tuple(packed()), TypeError),
    (packed(shape=torch.Size((3, 129))), ValueError),
    (packed(shape=torch.Size((4, 100))), ValueError),
    (packed(shape=torch.Size(())), ValueError),
    (packed(dtype=torch.float32), ValueError),
    (packed(dtype=torch.float64), ValueError),
    (packed(codes=torch.zeros(3, 128)), ValueError),
    (packed(codes=torch.zeros(3, 256, dtype=torch.uint8)[:, ::2]), ValueError),
    (packed(codes=torch.zeros(128, dtype=torch.uint8).expand(3, 128)), ValueError),
    (packed(ranges=torch.zeros(3, 2)), ValueError),
    (packed(ranges=torch.zeros(3, 2, 2, dtype=torch.int32)), ValueError),
])
def test_unpack8_refuses(p, exc):
    with pytest.raises(exc):
        fa.unpack8(p)


@pytest.mark.parametrize("name", ["x", "residual", "weight", "bias"])
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as fw
    t = dict(x=torch.ones(3, 8), residual=torch.ones(3, 8), weight=torch.ones(8),
             bias=torch.ones(8))
    with fw.dual_level():
        t[name] = fw.make_dual(t[name], torch.ones(t[name].shape))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fa.layer_norm(**t)
        if name == "x":
            with pytest.raises(RuntimeError, match="forward-mode"):
                fa.gelu8(t["x"])
            with pytest.raises(RuntimeError, match="forward-mode"):
                fa.linear8(t["x"], torch.ones(5, 8))


def test_structure_matches_the_header():
    assert ctypes.sizeof(_cabi.fa_norm) == 16 + 8 + 8 + 4 * 8 + 5 * 8
    assert len(block._NORM(3, 3, 1, 1, 0, 0.0, *[0] * 9)) == ctypes.sizeof(_cabi.fa_norm)
    assert ctypes.sizeof(_cabi.fa_linear8) == 16 + 8 + 3 * 16 + 7 * 8
    assert len(block._LINEAR(*[0] * 18)) == ctypes.sizeof(_cabi.fa_linear8)


def test_c_entries_refuse_before_any_launch():
    L = _cabi.load()
    size = ctypes.c_size_t(0)
    F32, F16 = 3, 1
    # dtype, shape, null and misaligned buffers
    for args, want in ((((16, 8, 4, 3, 8, 16, 16)), 1), ((16, 8, F32, 0, 8, 16, 16), 2),
                       ((16, 8, F32, 3, 0, 16, 16), 2), ((None, 8, F32, 3, 8, 16, 16), 5),
                       ((16, 8, F32, 3, 8, None, 16), 5), ((16, 8, F32, 3, 8, 16, None), 5),
                       ((18, 8, F32, 3, 8, 16, 16), 5), ((17, 8, F16, 3, 8, 16, 16), 5),
                       ((16, 8, F32, 3, 8, 24, 16), 5), ((16, 8, F32, 3, 8, 16, 20), 5)):
        assert L.fa_b200_pack8(*args, 0, None) == want, args
    assert L.fa_b200_unpack8(16, 16, F32, 3, 8, None, 8, 0, None) == 5
    assert L.fa_b200_unpack8(None, 16, F32, 3, 8, 16, 8, 0, None) == 5
    assert L.fa_b200_gelu8(16, 8, F32, 3, 8, 0, None, None, None, 0, None) == 5
    assert L.fa_b200_gelu8(16, 8, F32, 3, 8, 0, 16, 16, None, 0, None) == 5
    assert L.fa_b200_gelu8_backward(16, 8, None, 16, F32, 3, 8, 0, 16, 0, None) == 5
    assert L.fa_b200_gelu8_backward(16, 8, 16, 16, 0, 3, 8, 0, 16, 0, None) == 1

    def norm(**kw):
        f = dict(dtype=F32, weight_dtype=F32, rows=3, width=8, eps=1e-5, x=16, x_stride=8, stats=16)
        f.update(kw)
        return ctypes.byref(_cabi.fa_norm(**f))
    for kw, want in (({"dtype": 4}, 1), ({"weight_dtype": F16}, 1), ({"rows": 0}, 2),
                     ({"width": 0}, 2), ({"width": (1 << 24) + 1}, 2), ({"eps": -1.0}, 5),
                     ({"eps": float("nan")}, 5), ({"x": None}, 5), ({"x": 18}, 5),
                     ({"weight": 18}, 5), ({"residual": 17}, 5), ({"codes": 16}, 5),
                     ({"codes": 8, "ranges": 16}, 5), ({"stats": 12}, 5)):
        assert L.fa_b200_layer_norm(norm(**kw), 16, None, 0, None) == want, kw
    assert L.fa_b200_layer_norm(None, 16, None, 0, None) == 5
    assert L.fa_b200_layer_norm(norm(), None, None, 0, None) == 5

    def grad(dw=None, ws=None, size=0, dy=16, **kw):
        return L.fa_b200_layer_norm_backward(norm(**kw), dy, 8, None, 0, 16, dw, None, ws, size, 0,
                                             None)
    assert grad(dy=None) == 5 and grad(stats=None) == 5 and grad(x=None) == 5
    assert grad(dw=16) == 5 and grad(dw=16, ws=16, size=4) == 5 and grad(dw=16, ws=24, size=1 << 20) == 5
    assert L.fa_b200_layer_norm_backward_workspace_bytes(3, 8, 0, ctypes.byref(size)) == 0
    assert size.value >= 2 * 8 * 4
    assert L.fa_b200_layer_norm_backward_workspace_bytes(0, 8, 0, ctypes.byref(size)) == 2
    assert L.fa_b200_layer_norm_backward_workspace_bytes(3, 8, 0, None) == 5

    def linear(**kw):
        f = dict(dtype=F16, inputs=8, outputs=8, rows=3, x=512, x_stride=8, weight=512,
                 weight_stride=8, y=512)
        f.update(kw)
        return ctypes.byref(_cabi.fa_linear8(**f))
    back = dict(x=None, y=None, dy=512, dy_stride=8, dx=512)
    q = L.fa_b200_linear8_workspace_bytes
    assert q(linear(), 0, ctypes.byref(size)) == 0 and q(linear(), 0, None) == 5
    assert q(None, 0, ctypes.byref(size)) == 5
    # an operand that TMA does not read is copied
    assert q(linear(inputs=7, x_stride=7, weight_stride=7), 0, ctypes.byref(size)) == 0
    assert size.value >= 2 * 256
    room = 1 << 30
    for kw, want in (({"dtype": 4}, 1), ({"rows": 0}, 2), ({"inputs": 0}, 2),
                     ({"outputs": 1 << 23}, 2), ({"rows": (1 << 27) + 1}, 2), ({"x": None}, 5),
                     ({"weight": None}, 5), ({"x": 513}, 5), ({"y": None}, 5), ({"codes": 512}, 5),
                     ({"codes": 520, "ranges": 512}, 5), ({"dx": 512, "dy": 512}, 5)):
        assert L.fa_b200_linear8(linear(**kw), 512, room, 0, None) == want, kw
    for kw, want in (({"dy": None}, 5), ({"weight": None}, 5), ({"dx": None}, 5),
                     ({"y": 512, "x": 512}, 5), ({"dweight": 512}, 5), ({"dy": 511}, 5)):
        assert L.fa_b200_linear8_backward(linear(**{**back, **kw}), 512, room, 0, None) == want, kw
    copied = linear(**{**back, "outputs": 7, "dy_stride": 7})
    assert L.fa_b200_linear8_backward(copied, None, 0, 0, None) == 5
    assert L.fa_b200_linear8_backward(copied, 512, 16, 0, None) == 5
    assert L.fa_b200_linear8_backward(copied, 520, room, 0, None) == 5


def test_arrivals_in_the_other_block_are_of_the_cluster():
    """An arrival without a scope orders nothing outside its own block, and neither does
    a wait: the products' pairs are two blocks."""
    csrc = Path(block.__file__).parent / "csrc"
    text = (csrc / "linear8.cu").read_text() + (csrc / "tensor.cuh").read_text()
    remote = re.findall(r"mbarrier\.arrive[\w.:]*shared::cluster[\w.:]*", text)
    assert remote and all(".cluster.shared::cluster" in a for a in remote), remote
    # the barriers with such arrivals: the stages that are written, the sums that are read
    product = (csrc / "linear8.cu").read_text()
    waits = re.findall(r"stage_wait(<\w+>)?\((&full\[s\], \(n / S\)|&tm_empty)", product)
    assert len(waits) == 5 and all(kind == "<true>" for kind, _ in waits), waits
    assert product.count("wait.parity.acquire.cluster.shared::cta") == 2


@pytest.mark.parametrize("dtype,most", [(1, 160 << 20), (2, 160 << 20), (3, 80 << 20)])
def test_the_products_workspace_does_not_grow_with_their_sums(dtype, most):
    """Sizes at which a float32 copy of the result for every 32768 terms takes gigabytes."""
    L = _cabi.load()
    size = ctypes.c_size_t(0)

    def workspace(rows, inputs, outputs, **which):
        p = _cabi.fa_linear8(dtype=dtype, inputs=inputs, outputs=outputs, rows=rows,
                             x_stride=inputs, dy_stride=outputs, weight_stride=inputs,
                             **{k: 1 << 20 for k in which})
        assert L.fa_b200_linear8_workspace_bytes(ctypes.byref(p), 0, ctypes.byref(size)) == 0
        return size.value

    grad = dict(dy=1, codes=1, ranges=1, dweight=1)
    for rows, inputs, outputs in ((131072, 4096, 128256), (1100000, 4096, 16384),
                                  (1 << 27, 4096, 4096), (1 << 27, 16, 24), (70000, 1024, 4096),
                                  (1 << 22, 512, 2048)):
        assert workspace(rows, inputs, outputs, **grad) <= most
    assert workspace(60000, 40000, 4096, x=1, weight=1, y=1) <= most
    assert workspace(60000, 4096, 40000, dy=1, weight=1, dx=1) <= most


def test_the_wait_hook_is_bounded():
    assert _cabi.load().fa_b200_linear8_wait_selftest(1_000_000_001, 0, None) == 5
