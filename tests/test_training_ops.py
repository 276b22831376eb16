"""The training-step operators' refusals, which need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import frame_analytics_b200 as fa
from frame_analytics_b200 import _cabi, optim
from frame_analytics_b200._cabi import fa_heads, fa_matrix, fa_qk_params


def qk(**kw):
    args = dict(q=torch.zeros(2, 3, 4, 16), k=torch.zeros(2, 3, 2, 16), cos=torch.zeros(5, 8),
                sin=torch.zeros(5, 8))
    args.update(kw)
    return fa.qk_norm_rotary(**args)


@pytest.mark.parametrize("kw,exc", [
    ({}, TypeError),                                             # not on the GPU
    ({"q": torch.zeros(3, 4, 16)}, ValueError),
    ({"q": torch.zeros(2, 3, 4, 16, dtype=torch.float64)}, TypeError),
    ({"k": torch.zeros(2, 3, 2, 16, dtype=torch.float16)}, ValueError),
    ({"k": torch.zeros(2, 4, 2, 16)}, ValueError),
    ({"k": torch.zeros(2, 3, 2, 8)}, ValueError),
    ({"k": torch.zeros(2, 3, 0, 16)}, ValueError),
    ({"q": torch.zeros(2, 3, 4, 514), "k": torch.zeros(2, 3, 2, 514)}, ValueError),
    ({"sin": None}, ValueError),
    ({"sin": torch.zeros(5, 7)}, ValueError),
    ({"cos": torch.zeros(5, 9), "sin": torch.zeros(5, 9)}, ValueError),
    ({"cos": torch.zeros(5, 8).half(), "sin": torch.zeros(5, 8).half()}, ValueError),
    ({"cos": torch.zeros(2, 8), "sin": torch.zeros(2, 8)}, ValueError),   # 3 tokens
    ({"positions": torch.zeros(3)}, TypeError),
    ({"positions": torch.zeros(4, dtype=torch.int64)}, ValueError),
    ({"positions": torch.zeros(3, dtype=torch.int64), "cos": None, "sin": None}, ValueError),
    ({"eps": -1.0}, ValueError),
    ({"eps": float("nan")}, ValueError),
    ({"q_weight": torch.ones(15)}, ValueError),
    ({"q_weight": torch.ones(2, 16)}, ValueError),
    ({"q_weight": torch.ones(16).half()}, TypeError),
    ({"q_weight": torch.ones(16), "k_weight": torch.ones(2, 16)}, ValueError),
])
def test_qk_norm_rotary_refuses(kw, exc):
    with pytest.raises(exc):
        qk(**kw)


@pytest.mark.parametrize("kw,exc", [
    ({"x": torch.zeros(4)}, ValueError),
    ({"x": torch.zeros(4, 4, dtype=torch.float64)}, TypeError),
    ({"x": torch.zeros(4, 4, dtype=torch.int32)}, TypeError),
    ({"x": torch.zeros(4, 4)}, TypeError),                       # not on the GPU
    ({"steps": 0}, ValueError),
    ({"steps": 33}, ValueError),
    ({"steps": 2.0}, ValueError),
    ({"coefficients": (1.0, 2.0)}, ValueError),
    ({"coefficients": 3.0}, ValueError),
    ({"coefficients": [(1.5, -0.5, 0.0)] * 4}, ValueError),      # five steps
    ({"coefficients": (float("nan"), 0.0, 0.0)}, ValueError),
    ({"coefficients": (10.0, 0.0, 0.0)}, ValueError),            # grows without bound
])
def test_orthogonalize_refuses(kw, exc):
    args = dict(x=torch.zeros(4, 6), steps=5, coefficients=optim.NEWTON_SCHULZ)
    args.update(kw)
    with pytest.raises(exc):
        fa.orthogonalize(**args)


def step(w=None, g=None, m=None, **kw):
    w = [torch.zeros(4, 6)] if w is None else w
    g = [torch.zeros_like(t) for t in w] if g is None else g
    m = [torch.zeros(t.shape) for t in w] if m is None else m
    fa.muon_step(w, g, m, **{"lr": 0.1, **kw})


@pytest.mark.parametrize("kw,exc", [
    ({}, TypeError),                                             # not on the GPU
    ({"g": []}, ValueError),
    ({"w": [torch.zeros(4)]}, ValueError),
    ({"w": [torch.zeros(4, 4), torch.zeros(4, 4).half()]}, TypeError),
    ({"g": [torch.zeros(6, 4)]}, ValueError),
    ({"g": [torch.zeros(4, 6).half()]}, ValueError),
    ({"m": [torch.zeros(4, 6).half()]}, ValueError),
    ({"lr": -1.0}, ValueError),
    ({"lr": float("inf")}, ValueError),
    ({"momentum": 1.0}, ValueError),
    ({"weight_decay": -0.1}, ValueError),
    ({"scale": "best"}, ValueError),
    ({"steps": 0}, ValueError),
])
def test_muon_step_refuses(kw, exc):
    with pytest.raises(exc):
        step(**kw)


def test_muon_step_of_nothing():
    fa.muon_step([], [], [], lr=0.1)


def test_muon_refuses_vectors_and_bad_settings():
    with pytest.raises(ValueError):
        fa.Muon([torch.nn.Parameter(torch.zeros(3))])
    for kw in ({"lr": -1.0}, {"momentum": 1.0}, {"weight_decay": -1.0}, {"scale": "x"},
               {"steps": 0}):
        with pytest.raises(ValueError):
            fa.Muon([torch.nn.Parameter(torch.zeros(3, 3))], **kw)


def test_c_entries_refuse_before_any_launch():
    L = _cabi.load()
    coef = (ctypes.c_double * 3)(1.5, -0.5, 0.0)
    size = ctypes.c_size_t(0)
    m = (fa_matrix * 1)((16, 16, None, 4, 6, 6, 6, 0.1))
    assert L.fa_b200_orthogonalize_workspace_bytes(m, 1, 3, ctypes.byref(size)) == 0
    assert size.value > 0
    assert L.fa_b200_orthogonalize_workspace_bytes(m, 1, 0, ctypes.byref(size)) == 1
    assert L.fa_b200_orthogonalize_workspace_bytes(None, 1, 3, ctypes.byref(size)) == 5
    assert L.fa_b200_orthogonalize(None, 1, 3, coef, 1, 16, 1 << 20, 0, None) == 5
    assert L.fa_b200_orthogonalize(m, 0, 3, coef, 1, 16, 1 << 20, 0, None) == 5
    assert L.fa_b200_orthogonalize(m, 1, 4, coef, 1, 16, 1 << 20, 0, None) == 1
    assert L.fa_b200_muon_step(m, 1, 3, coef, 1, 0.9, 1, 1.0, 16, 1 << 20, 0, None) == 5
    bad = (fa_matrix * 1)((16, 16, None, 0, 6, 6, 6, 0.1))
    assert L.fa_b200_orthogonalize(bad, 1, 3, coef, 1, 16, 1 << 20, 0, None) == 2
    narrow = (fa_matrix * 1)((16, 16, None, 4, 6, 5, 6, 0.1))
    assert L.fa_b200_orthogonalize(narrow, 1, 3, coef, 1, 16, 1 << 20, 0, None) == 2
    assert L.fa_b200_qk_norm_rotary_backward_workspace_bytes(1, 1, 1, 0, 8,
                                                             ctypes.byref(size)) == 2


def test_structures_match_the_header():
    assert ctypes.sizeof(fa_heads) == 40
    assert ctypes.sizeof(fa_matrix) == 56
    assert ctypes.sizeof(fa_qk_params) == 40 + 24 + 16 + 16 + 8


def test_the_wait_limit_is_at_most_the_default():
    L = _cabi.load()
    assert L.fa_b200_orthogonalize_wait_limit(2_000_000_001) == 5
    assert L.fa_b200_orthogonalize_wait_limit(1_000_000) == 0
    assert L.fa_b200_orthogonalize_wait_limit(0) == 0


def workspace(shapes, dtype):
    L = _cabi.load()
    m = (fa_matrix * len(shapes))(*[(16, 16, None, r, c, c, c, 0.1) for r, c in shapes])
    size = ctypes.c_size_t(0)
    assert L.fa_b200_orthogonalize_workspace_bytes(m, len(shapes), dtype, ctypes.byref(size)) == 0
    return size.value


@pytest.mark.parametrize("code", [1, 2, 3], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("shapes", [
    [(4096, 4096)] * 128,
    [(4096, 11008), (11008, 4096), (4096, 4096)] * 32,
    [(16, 16)] + [(2048, 2048)] * 200 + [(8192, 8192)],
])
def test_workspace_does_not_grow_with_the_list(shapes, code):
    one = max(workspace([s], code) for s in set(shapes))
    assert one <= workspace(shapes, code) <= max(one, (2 << 30) + (16 << 20))


@pytest.mark.parametrize("which", ["cos", "sin"])
def test_qk_norm_rotary_refuses_tables_that_want_a_gradient(which):
    table = torch.zeros(5, 8, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        qk(**{which: table})
    with pytest.raises(ValueError, match="no gradient"):  # computed from learned frequencies
        qk(**{which: 2 * table})
    with torch.no_grad(), pytest.raises(TypeError):  # the next check: not on the GPU
        qk(**{which: table})


@pytest.mark.parametrize("which", ["q", "k", "cos", "sin", "q_weight", "k_weight"])
def test_qk_norm_rotary_refuses_forward_mode(which):
    import torch.autograd.forward_ad as fw
    shapes = dict(q=(2, 3, 4, 16), k=(2, 3, 2, 16), cos=(5, 8), sin=(5, 8), q_weight=(16,),
                  k_weight=(16,))
    t = {n: torch.ones(s) for n, s in shapes.items()}
    with fw.dual_level():
        with pytest.raises(TypeError):  # no tangent: the next check, not on the GPU
            qk(**t)
        t[which] = fw.make_dual(t[which], torch.ones(shapes[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            qk(**t)


@pytest.mark.parametrize("shape", [(32769, 32769), (2, 32769, 40000), (1, (1 << 22) + 1),
                                   (1 << 33, 4)])
def test_matrices_past_the_limits_are_refused_before_anything_is_allocated(shape):
    x = torch.zeros(1).expand(shape)
    with pytest.raises(ValueError, match="at most"):
        fa.orthogonalize(x)
    with pytest.raises(ValueError, match="at most"):
        fa.muon_step([x], [x], [x], lr=0.1)
    L = _cabi.load()
    size = ctypes.c_size_t(0)
    m = (fa_matrix * 1)((16, 16, None, 32769, 32769, 32769, 32769, 0.1))
    assert L.fa_b200_orthogonalize_workspace_bytes(m, 1, 3, ctypes.byref(size)) == 2
    m[0].rows, m[0].cols = 1, (1 << 22) + 1
    assert L.fa_b200_orthogonalize_workspace_bytes(m, 1, 3, ctypes.byref(size)) == 2


def test_qk_norm_rotary_looks_at_eps_in_every_call():
    eps = torch.tensor(1e-6)
    with pytest.raises(TypeError):  # not on the GPU
        qk(eps=eps)
    with pytest.raises(ValueError, match="eps"):
        qk(eps=eps.fill_(-1.0))


def test_the_example_starts_from_anywhere(tmp_path):
    import os
    import subprocess
    import sys

    from conftest import REPO
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    run = subprocess.run([sys.executable, str(REPO / "examples" / "train_restoration.py"), "--help"],
                         cwd=tmp_path, env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert "--steps" in run.stdout


def test_waits_for_the_pairs_other_block_are_of_the_cluster():
    """Barriers at which threads of the other block arrive, or its copies: the sums that
    are read, and the stages."""
    import re
    from pathlib import Path
    csrc = Path(fa.__file__).parent / "csrc"
    waits = re.findall(r"wait_bar(<\w+>)?\((&full\[s\]|&tm_empty|&sm_empty)",
                       (csrc / "orthogonalize.cu").read_text())
    assert len(waits) == 3 and all(kind == "<PAIR>" for kind, _ in waits), waits
    assert "try_wait.parity.acquire.cluster.shared::cta" in (csrc / "tensor.cuh").read_text()
