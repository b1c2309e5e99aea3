"""What the orthogonalised step refuses, on the host and before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch


def _muon(**kw):
    from engraft_ngram_amd import _lib
    one = (ctypes.c_void_p * 1)(256)
    coef = (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315)
    o = _lib.EgMuon()
    o.rows, o.cols, o.count, o.planes = 100, 200, 1, 2
    o.params = o.grads = o.momenta = ctypes.cast(one, ctypes.c_void_p)
    o.coefficients, o.steps = ctypes.cast(coef, ctypes.c_void_p), 1
    o.momentum, o.eps, o.keep, o.rate = 0.9, 1e-7, 1.0, 0.1
    o._kept = (one, coef)
    for k, x in kw.items():
        setattr(o, k, x)
    return o


@pytest.mark.parametrize("needle,bad", [
    ("0 x 200", dict(rows=0)), ("2^20", dict(cols=(1 << 20) + 1)), ("count=-1", dict(count=-1)),
    ("NULL", dict(params=None)), ("planes=3", dict(planes=3)), ("dtype=9", dict(grad_dtype=9)),
    ("steps=0", dict(steps=0)), ("steps=101", dict(steps=101)), ("eps=0", dict(eps=0.0)),
    ("not finite", dict(rate=float("nan"))),
])
def test_arguments_are_checked(needle, bad):
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    o = _muon(**bad)
    rc = lib.eg_muon_step(ctypes.byref(o), 256, 1 << 40, None)
    assert rc == _lib.EG_ERR_ARG and needle in lib.eg_last_error().decode()


def test_workspace_is_checked():
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    need = lib.eg_muon_workspace_size(100, 200, 1, 2)
    assert need > 0 and lib.eg_muon_workspace_size(100, 200, 2, 2) > need > lib.eg_muon_workspace_size(100, 200, 1, 1)
    assert lib.eg_muon_workspace_size(100, 200, 1, 3) == -1
    o = _muon()
    assert lib.eg_muon_step(ctypes.byref(o), 256, need - 1, None) == _lib.EG_ERR_WORKSPACE
    assert lib.eg_muon_step(ctypes.byref(o), 8, need, None) == _lib.EG_ERR_ARG
    o = _muon(count=0)
    assert lib.eg_muon_step(ctypes.byref(o), None, 0, None) == _lib.EG_OK
    # a NULL among the matrices
    none = (ctypes.c_void_p * 1)(None)
    o = _muon(grads=ctypes.cast(none, ctypes.c_void_p))
    assert lib.eg_muon_step(ctypes.byref(o), 256, need, None) == _lib.EG_ERR_ARG


def test_coefficients_that_leave_the_range():
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    coef = (ctypes.c_float * 6)(100.0, 0.0, 0.0, 1.0, 0.0, 0.0)  # singular values of up to 100 after a step
    o = _muon(coefficients=ctypes.cast(coef, ctypes.c_void_p), steps=2)
    assert lib.eg_muon_step(ctypes.byref(o), 256, 1 << 40, None) == _lib.EG_ERR_ARG
    assert "singular values" in lib.eg_last_error().decode()


def test_host_tensors_are_refused():
    from engraft_ngram_amd import muon
    w = torch.zeros((3, 4))
    with pytest.raises(ValueError, match="on the GPU"):
        muon.muon_step([w], [w], [w], lr=0.1)
    with pytest.raises(ValueError, match="on the GPU"):
        muon.orthogonalize(w)
    with pytest.raises(ValueError, match="on the GPU"):
        muon.MuonState([w])


def test_check_says_what_a_step_would():
    """eg_muon_check refuses what eg_muon_step refuses, and launches nothing."""
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    for bad in (dict(rows=0), dict(cols=(1 << 20) + 1), dict(planes=3), dict(rate=float("inf"))):
        o = _muon(**bad)
        said = [(f(ctypes.byref(o), *rest), lib.eg_last_error()) for f, rest in
                ((lib.eg_muon_check, ()), (lib.eg_muon_step, (256, 1 << 40, None)))]
        assert said[0] == said[1] and said[0][0] == _lib.EG_ERR_ARG
    assert lib.eg_muon_check(ctypes.byref(_muon(count=0))) == _lib.EG_OK


@pytest.mark.parametrize("what,param,grad,momentum", [
    ("params of matrix 0 overlap themselves", [(0, 3, 5), (4096, 4, 1)], 1 << 20, 1 << 21),
    ("params of matrix 0 overlap params of matrix 1", [(0, 4, 1), (12, 4, 1)], 1 << 20, 1 << 21),
    ("params of matrix 0 overlap params of matrix 1", [(0, 4, 1), (0, 4, 1)], 1 << 20, 1 << 21),
    ("grads of matrix 0 overlap params of matrix 1", [(0, 4, 1), ((1 << 18) + 1, 4, 1)], 1 << 18, 1 << 21),
    ("momenta", [(0, 4, 1), (1 << 18, 4, 1)], 1 << 20, 1 << 20),
])
def test_overlaps_are_refused(what, param, grad, momentum):
    """Matrices of 6 x 4 f32 at element offsets and strides; gradients and momenta lie one after the other."""
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    base = 1 << 30
    for (a, row, col), (b, _, _) in [param]:
        o = _muon(rows=6, cols=4, count=2)
        lists = [(ctypes.c_void_p * 2)(base + 4 * x, base + 4 * y) for x, y in
                 ((a, b), (grad, grad + 24), (momentum, momentum + 24))]
        o.params, o.grads, o.momenta = (ctypes.cast(x, ctypes.c_void_p) for x in lists)
        o.param_stride[:] = [row, col]
        o.grad_stride[:] = o.momentum_stride[:] = [4, 1]
        assert lib.eg_muon_check(ctypes.byref(o)) == _lib.EG_ERR_ARG
        assert what in lib.eg_last_error().decode(), lib.eg_last_error()
        assert lib.eg_muon_step(ctypes.byref(o), 256, 1 << 40, None) == _lib.EG_ERR_ARG


def test_what_lies_apart_is_taken():
    """Columns of one buffer, rows between rows, a gradient in its own weight's place."""
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    base = 1 << 30
    for params, grads, stride in (((0, 4), (1 << 20, 1 << 20), (8, 1)), ((0, 8), (1 << 20, 1 << 20), (16, 1)),
                                  ((0, 24), (0, 24), (4, 1)), ((0, 6), (0, 6), (1, 12)), ((0, 1), (1 << 20, 1 << 20), (8, 2))):
        o = _muon(rows=6, cols=4, count=2)
        lists = [(ctypes.c_void_p * 2)(*(base + 4 * x for x in at)) for at in (params, grads, (1 << 24, (1 << 24) + 24))]
        o.params, o.grads, o.momenta = (ctypes.cast(x, ctypes.c_void_p) for x in lists)
        o.param_stride[:] = o.grad_stride[:] = list(stride)
        o.momentum_stride[:] = [4, 1]
        assert lib.eg_muon_check(ctypes.byref(o)) == _lib.EG_OK, (params, lib.eg_last_error())


def test_workspace_does_not_grow_with_every_matrix():
    """Many large matrices share at most 2 GiB; one alone takes what it needs, whatever that is."""
    from engraft_ngram_amd import _lib
    size = _lib.load().eg_muon_workspace_size
    for planes in (1, 2):
        for rows, cols in ((2560, 2560), (4096, 4096), (10_240, 2560), (20_000, 20_000)):
            one = size(rows, cols, 1, planes)
            assert one <= size(rows, cols, 64, planes) <= max(one, 2 << 30)
            assert size(rows, cols, 1000, planes) == size(rows, cols, 64, planes)
    assert size(64, 256, 64, 2) > 60 * (size(64, 256, 2, 2) - size(64, 256, 1, 2))
