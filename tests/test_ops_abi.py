"""CPU: argument checks of the batched operators (include/mplc_hip_ops.h) - every refusal comes before any HIP call."""
import ctypes
import os
import re

import pytest
import torch

from mplc import _native, dense, muon

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E_ARG, E_WS, E_SHAPE = -1, -2, -3
BUF = (ctypes.c_double * 64)()
P = ctypes.addressof(BUF) // 16 * 16 + 16


def dense_t(**kw):
    t = dense.DenseT()
    t.n_models, t.rows, t.in_, t.out = 2, 3, 4, 5
    t.x = t.w = t.y = t.dy = t.dx = t.dw = t.db = P
    t.x_ld, t.w_ld, t.y_ld, t.dy_ld, t.dx_ld, t.dw_ld = 4, 5, 5, 5, 4, 5
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def muon_t(**kw):
    t = muon.MuonT()
    t.n_models, t.rows, t.cols, t.steps = 2, 400, 70, 5
    t.a, t.b, t.c = muon.COEFFICIENTS
    t.g = t.out = t.m = t.w = t.workspace = P
    t.g_ld = t.out_ld = t.m_ld = t.w_ld = 70
    t.workspace_bytes = 1 << 40
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def test_structs_match_the_library():
    q = _native.lib().mplc_ops_layout
    assert q(0) == ctypes.sizeof(dense.DenseT) and q(1) == ctypes.sizeof(muon.MuonT) and q(2) == -1 and q(-1) == -1
    text = open(os.path.join(REPO, "include", "mplc_hip_ops.h")).read()
    for name, host in (("mplc_dense_t", dense.DenseT), ("mplc_muon_t", muon.MuonT)):
        body = re.sub(r"/\*.*?\*/", "", text[:text.index("} " + name)], flags=re.S).split("typedef struct {")[-1]
        fields = [re.sub(r"[\s*]", "", f.split()[-1] if i == 0 else f)
                  for line in body.split(";") if line.strip() for i, f in enumerate(line.split(","))]
        assert [f.rstrip("_") for f, _ in host._fields_] == fields
    for k, v in dense.ACTIVATIONS.items():
        assert re.search(rf"#define MPLC_ACT_{k.upper()} {v}\b", text)


def test_dense_argument_errors():
    lib = dense._lib()
    fwd = lambda **kw: lib.mplc_dense_forward(ctypes.byref(dense_t(**kw)), None)  # noqa: E731
    bwd = lambda **kw: lib.mplc_dense_backward(ctypes.byref(dense_t(**kw)), None)  # noqa: E731
    assert lib.mplc_dense_forward(None, None) == E_ARG and lib.mplc_dense_backward(None, None) == E_ARG
    for f in (fwd, bwd):
        for kw in ({"n_models": -1}, {"n_models": 65536}, {"rows": -1}, {"in_": 0}, {"out": 0}, {"dtype": 3},
                   {"dtype": -1}, {"activation": 4}, {"activation": -1}, {"w": None}, {"w_ld": 4}, {"x": None},
                   {"x_ld": 3}, {"workspace": P + 8}):
            assert f(**kw) == E_ARG, kw
    for kw in ({"y": None}, {"y_ld": 4}, {"residual": P, "residual_ld": 4}, {"z": P, "z_ld": 1}):
        assert fwd(**kw) == E_ARG, kw
    for kw in ({"dy": None}, {"dy_ld": 4}, {"activation": 2}, {"activation": 1, "z": P, "z_ld": 2}, {"dx_ld": 3},
               {"dw_ld": 4}):
        assert bwd(**kw) == E_ARG, kw
    assert fwd(n_models=0) == 0 and fwd(rows=0) == 0 and bwd(n_models=0, dx=None) == 0
    assert bwd(n_models=0, x_shared=1) == E_SHAPE  # the sum over no models
    big = dict(rows=3, in_=9216, out=8, x_ld=9216, w_ld=8, y_ld=8)  # a split sum needs its workspace
    n = lib.mplc_dense_forward_workspace_bytes(ctypes.byref(dense_t(**big)))
    assert n > 0 and fwd(**big) == E_WS and fwd(workspace=P, workspace_bytes=n - 1, **big) == E_WS
    act = dict(activation=3, z=P, z_ld=5)
    n = lib.mplc_dense_backward_workspace_bytes(ctypes.byref(dense_t(**act)))
    assert n > 0 and bwd(**act) == E_WS and bwd(workspace=P, workspace_bytes=n - 1, **act) == E_WS
    huge = dict(n_models=60000, rows=1 << 20, in_=1 << 20, out=1 << 20, x_ld=1 << 20, w_ld=1 << 20, y_ld=1 << 20)
    assert fwd(**huge) == E_SHAPE


def test_muon_argument_errors():
    lib = muon._lib()
    for f in (lib.mplc_orthogonalize, lib.mplc_muon_step):
        assert f(None, None) == E_ARG
        for kw in ({"n_models": -1}, {"n_models": 65536}, {"rows": 0}, {"cols": 0}, {"dtype": 3}, {"steps": 0},
                   {"steps": 17}, {"a": 4.0, "b": -4.0, "c": 3.0}, {"a": float("nan")}, {"c": float("inf")}, {"g": None},
                   {"g_ld": 69}, {"workspace": P + 4}):
            assert f(ctypes.byref(muon_t(**kw)), None) == E_ARG, kw
        assert f(ctypes.byref(muon_t(workspace_bytes=16)), None) == E_WS
        assert f(ctypes.byref(muon_t(workspace=None)), None) == E_WS
        assert f(ctypes.byref(muon_t(n_models=0)), None) == 0
    for kw in ({"out": None}, {"out_ld": 69}):
        assert lib.mplc_orthogonalize(ctypes.byref(muon_t(**kw)), None) == E_ARG
    for kw in ({"m": None}, {"w": None}, {"m_ld": 69}, {"w_ld": 69}):
        assert lib.mplc_muon_step(ctypes.byref(muon_t(**kw)), None) == E_ARG


def test_workspace_sizes_follow_the_sizes():
    lib = muon._lib()
    size = lambda **kw: lib.mplc_muon_step_workspace_bytes(ctypes.byref(muon_t(**kw)))  # noqa: E731
    assert size(rows=0) == 0 and 0 < size() < size(n_models=20) and size(rows=65, cols=4000) > 65 * 4000 * 4 and size(rows=9, cols=32) == 0


def test_singular_range():
    assert muon.singular_range(5, muon.COEFFICIENTS) < 1.21
    assert muon.singular_range(9, (1.5, -0.5, 0.0)) == 1.0
    assert muon.singular_range(3, (2.5, 0.0, 0.0)) > 2.0
    assert muon.update_scale(128, 10) == 1.0 and muon.update_scale(10, 40) == 2.0


def test_host_checks_refuse_cpu_tensors():
    x, w = torch.zeros(2, 3, 4), torch.zeros(2, 4, 5)
    for f in (lambda: dense.dense_forward(x, w), lambda: dense.dense_backward(torch.zeros(2, 3, 5), x, w),
              lambda: muon.orthogonalize(w), lambda: muon.muon_step(w, w, w, lr=0.1)):
        with pytest.raises(ValueError, match="CUDA"):
            f()
    for f in (lambda: dense.dense_forward(None, w), lambda: muon.orthogonalize([1.0])):
        with pytest.raises(TypeError):
            f()


def test_memory_overlap_checks():
    def check(out, other, same=()):
        ts = (out, other)
        dense._no_overlap(ts, ("out", "other"), [t.data_ptr() for t in ts], [dense._span(t) for t in ts], [0], [1], same)
    rows = torch.zeros(3, 100)
    a, b, c = (rows[:, o:o + 12].view(3, 3, 4) for o in (0, 12, 20))
    check(a, b)
    check(a, a, same=((0, 1),))
    for p, q in ((a, a), (b, c), (a, rows)):
        with pytest.raises(ValueError, match="share memory"):
            check(p, q)
    with pytest.raises(ValueError, match="share memory"):
        check(b, c, same=((0, 1),))
    dense._writable(a, "a")
    dense._writable(torch.zeros(5, 3, 4).transpose(0, 1), "beside")
    for t in (torch.zeros(1, 3, 4).expand(2, 3, 4), torch.zeros(40).as_strided((2, 3, 4), (6, 5, 1))):
        with pytest.raises(ValueError, match="overlap"):
            dense._writable(t, "t")
