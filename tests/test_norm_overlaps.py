"""Memory that the norm and its gradients write and must not share with what they read or write besides, refused on the host and
before any launch."""
from __future__ import annotations

import ctypes

import pytest

from tests.test_fp8_arguments import _lib, _matrix, _norm, _norm_grad, _ref, _refused

MB = 1 << 20  # x, the residual and the weight are at 1, 2 and 3 of them, 5 x 300 f32 each; h is at 4, y at 5


def _run(rstd=6 * MB, y=5 * MB, y8=None, h=4 * MB, **kw):
    return _lib().load().eg_add_rms_norm(ctypes.byref(_norm(**kw)), h, 300, y, 0, 300, _ref(y8), rstd, None)


@pytest.mark.parametrize("at,name", [(1, "x"), (2, "the residual"), (3, "the weight"), (4, "h"), (5, "y")])
def test_rstd(at, name):
    for to in (at * MB, at * MB + 1196, at * MB - 16):
        with_y = _run(rstd=to)
        said = _lib().load().eg_last_error().decode()
        assert with_y == _lib().EG_ERR_ARG and "rstd" in said and name in said and "overlaps" in said, said


@pytest.mark.parametrize("at,name", [(1, "x"), (2, "the residual"), (3, "the weight"), (4, "h"), (6, "rstd")])
def test_scales(at, name):
    """5 rows of 300 values: 3 scales and their fill each."""
    for to in (at * MB, at * MB - 16, at * MB + 16):
        rc = _run(y=None, y8=_matrix(5, 300, q=5 * MB, scales=to))
        said = _lib().load().eg_last_error().decode()
        assert rc == _lib().EG_ERR_ARG and "y's scales" in said and name in said and "overlaps" in said, said


def test_scales_on_their_blocks():
    _refused(_run(y=None, y8=_matrix(5, 300, q=5 * MB, scales=5 * MB + 4 * 384)), "overlaps")


def test_the_weight():
    _refused(_run(y=3 * MB + 1196), "y overlaps the weight")
    _refused(_run(h=3 * MB + 1196), "h overlaps the weight")
    _refused(_run(y=None, y8=_matrix(5, 300, q=3 * MB + 16)), "y overlaps the weight")
    _refused(_run(rstd=3 * MB, residual=None, h=None), "rstd overlaps the weight")


# d_y, h, the weight and rstd are at 1, 2, 3 and 4 of them
@pytest.mark.parametrize("what,at,needle", [
    ("d_x2", 6 * MB, "d_x overlaps d_x2"), ("d_x2", 6 * MB + 5996, "overlaps"), ("d_x", 3 * MB, "overlaps the weight"),
    ("d_x", 4 * MB + 16, "overlaps rstd"), ("d_x2", 4 * MB - 5996, "overlaps rstd"),
    ("d_weight", 1 * MB, "overlaps d_y"), ("d_weight", 2 * MB + 5996, "overlaps h"), ("d_weight", 3 * MB, "overlaps the weight"),
    ("d_weight", 4 * MB + 16, "overlaps rstd"), ("d_weight", 6 * MB, "d_x overlaps"), ("d_weight", 5 * MB, "overlaps d_residual"),
    ("ws", 1 * MB, "the workspace overlaps d_y"), ("ws", 2 * MB, "the workspace overlaps h"), ("ws", 3 * MB, "the workspace overlaps the weight"),
    ("ws", 4 * MB, "the workspace overlaps rstd"), ("ws", 6 * MB, "overlaps the workspace"), ("ws", 7 * MB, "overlaps the workspace"),
    ("ws", 5 * MB, "the workspace overlaps d_residual"),
])
def test_gradients(what, at, needle):
    lib = _lib().load()
    o = _norm_grad(d_residual=5 * MB, dr_stride=300)
    to = {"d_x": 6 * MB, "d_x2": None, "d_weight": 7 * MB, "ws": 8 * MB, what: at}
    _refused(lib.eg_add_rms_norm_grad(ctypes.byref(o), to["d_x"], 0, 300, to["d_x2"], 0, 300, to["d_weight"], to["ws"],
                                      lib.eg_add_rms_norm_grad_workspace_size(5, 300), None), needle)
