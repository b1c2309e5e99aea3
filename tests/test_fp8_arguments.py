"""What the 8-bit products, the norms and the clipping refuse, on the host and before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch


def _lib():
    from engraft_ngram_amd import _lib
    return _lib


def _matrix(rows, k, block_rows=1, **kw):
    lib = _lib()
    m = lib.EgFp8Matrix()
    blocks = (k + 127) // 128
    m.q, m.scales, m.rows, m.k, m.block_rows = 4096, 4096, rows, k, block_rows
    m.stride, m.scale_stride = blocks * 128, (blocks + 3) // 4 * 4
    for name, x in kw.items():
        setattr(m, name, x)
    return m


def _ref(m):
    return None if m is None else ctypes.byref(m)


def _refused(rc, needle, code=None):
    lib = _lib()
    said = lib.load().eg_last_error().decode()
    assert rc == (lib.EG_ERR_ARG if code is None else code) and needle in said, (rc, said)


@pytest.mark.parametrize("needle,bad", [
    ("rows in", dict(rows=-1)), ("rows in", dict(k=0)), ("rows in", dict(k=(1 << 22) + 1)), ("stride=256", dict(stride=256)),
    ("stride=392", dict(stride=392)), ("scale_stride=6", dict(scale_stride=6)), ("NULL", dict(q=None)), ("NULL", dict(scales=None)),
    ("aligned", dict(q=4100)), ("aligned", dict(scales=4098)), ("a scale covers 128 rows", dict(block_rows=128)),
])
def test_matrices_are_checked(needle, bad):
    lib = _lib().load()
    a, w = _matrix(5, 300), _matrix(7, 300, 128)
    for name, x in bad.items():
        setattr(a, name, x)
    _refused(lib.eg_fp8_product(_ref(a), _ref(w), None, 4096, 7, None, 0, 0, None, 0, None), needle)
    _refused(lib.eg_fp8_quantize(4096, 0, 300, _ref(a), None), needle)


@pytest.mark.parametrize("needle,args", [
    ("NULL matrix", dict(b=None)), ("k=300, b 301", dict(b="k")), ("rows of 7 outputs", dict(ldc=6)),
    ("NULL output", dict(c=None)), ("dtype=5", dict(dtype=5)), ("misaligned output", dict(c=4097)),
])
def test_products_are_checked(needle, args):
    lib = _lib().load()
    b = {"k": _matrix(7, 301, 128), None: None, 0: _matrix(7, 300, 128)}[args.get("b", 0)]
    _refused(lib.eg_fp8_product(_ref(_matrix(5, 300)), _ref(b), None, args.get("c", 4096), args.get("ldc", 7), None, 0,
                                args.get("dtype", 0), None, 0, None), needle)


def test_linear_is_checked():
    lib = _lib().load()
    w = _matrix(7, 300, 128)
    size = lib.eg_fp8_linear_workspace_size
    assert size(1, 7, 0, 300) == 0 and size(100, 7, 0, 300) == 100 * (384 + 4) and size(-1, 7, 0, 300) == -1 and size(5, 7, 0, 0) == -1
    assert size(100, 7, 5, 10_240) > 100 * (10_240 + 80) and lib.eg_fp8_product_workspace_size(100, 7, 5, 10_240) > 0
    assert lib.eg_fp8_product_workspace_size(1, 7, 0, 10_240) == 0 and lib.eg_fp8_product_workspace_size(1, -7, 0, 10_240) == -1
    a, b = _matrix(100, 10_240), _matrix(7, 10_240, 128)
    _refused(lib.eg_fp8_product(_ref(a), _ref(b), None, 4096, 7, None, 0, 0, 4096, 100, None), "workspace", _lib().EG_ERR_WORKSPACE)
    run = lambda x=4096, dtype=0, m=100, ld=300, ws=4096, n=1 << 20: lib.eg_fp8_linear(  # noqa: E731
        x, dtype, m, ld, _ref(w), None, 4096, 7, None, 0, 0, ws, n, None)
    _refused(run(x=None), "NULL")
    _refused(run(x=4098), "misaligned")
    _refused(run(dtype=3), "dtype=3")
    _refused(run(m=-1), "rows")
    _refused(run(ld=299), "apart")
    _refused(run(n=100), "workspace", _lib().EG_ERR_WORKSPACE)
    _refused(run(ws=None), "aligned")
    _refused(run(ws=4104), "aligned")
    assert run(m=0, x=None, ws=None, n=0) == 0


def test_weights_are_checked():
    lib = _lib().load()
    w, t = _matrix(7, 300, 128), _matrix(300, 8, 128)
    _refused(lib.eg_fp8_quantize_weight(4096, 0, 300, 1, _ref(w), _ref(t), None), "the transpose of 7 x 300")
    _refused(lib.eg_fp8_quantize_weight(None, 0, 300, 1, _ref(w), None, None), "NULL")
    _refused(lib.eg_fp8_quantize_weight(4096, 7, 300, 1, _ref(w), None, None), "dtype=7")
    _refused(lib.eg_fp8_dequantize(_ref(w), 4096, 0, 299, None), "apart")
    _refused(lib.eg_fp8_dequantize(None, 4096, 0, 300, None), "NULL")


def _norm(**kw):
    o = _lib().EgNorm()
    o.x, o.residual, o.weight, o.rows, o.d, o.x_stride, o.r_stride, o.eps = 1 << 20, 2 << 20, 3 << 20, 5, 300, 300, 300, 1e-6
    for name, x in kw.items():
        setattr(o, name, x)
    return o


def _run_norm(o, h=4 << 20, y=5 << 20, y_dtype=0, y8=None, h_stride=300, y_stride=300):
    return _lib().load().eg_add_rms_norm(ctypes.byref(o), h, h_stride, y, y_dtype, y_stride, _ref(y8), None, None)


@pytest.mark.parametrize("needle,kw,more", [
    ("-1 rows", dict(rows=-1), {}), ("5 rows of 0", dict(d=0), {}), ("eps", dict(eps=-1.0), {}), ("eps", dict(eps=float("nan")), {}),
    ("x: NULL", dict(x=None), {}), ("x: dtype=4", dict(x_dtype=4), {}), ("x: rows", dict(x_stride=299), {}), ("residual: rows", dict(r_stride=10), {}),
    ("x's type or f32", dict(x_dtype=0, r_dtype=1), {}), ("misaligned weight", dict(weight=4097), {}),
    ("h: NULL", {}, dict(h=None)), ("y or y8", {}, dict(y=None)), ("y overlaps x", {}, dict(y=(1 << 20) + 40)),
    ("y overlaps h", {}, dict(y=(4 << 20) + 40)), ("h overlaps x", {}, dict(h=(1 << 20) + 40)), ("h overlaps the residual", {}, dict(h=(2 << 20) + 1200)),
    ("y overlaps the residual", {}, dict(y=(2 << 20) + 400)), ("y: misaligned", {}, dict(y=(5 << 20) + 2)),
])
def test_norms_are_checked(needle, kw, more):
    _refused(_run_norm(_norm(**kw), **more), needle)


def test_norms_in_blocks_are_checked():
    _refused(_run_norm(_norm(), y=None, y8=_matrix(5, 301)), "y8 is 5 x 301")
    _refused(_run_norm(_norm(), y8=_matrix(5, 300)), "y or y8")
    _refused(_run_norm(_norm(), y=None, y8=_matrix(5, 300, q=1 << 20)), "y overlaps x")
    _refused(_run_norm(_norm(d=20_481, x_stride=50_000, r_stride=50_000), h_stride=50_000, y_stride=50_000), "at most 20480", _lib().EG_ERR_UNSUPPORTED)
    assert _run_norm(_norm(rows=0, x=None, residual=None), h=None) == 0


def _norm_grad(**kw):
    o = _lib().EgNormGrad()
    o.d_y, o.h, o.weight, o.rstd, o.rows, o.d, o.dy_stride, o.h_stride = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5, 300, 300, 300
    for name, x in kw.items():
        setattr(o, name, x)
    return o


@pytest.mark.parametrize("needle,kw,more", [
    ("d_y: NULL", dict(d_y=None), {}), ("h: dtype", dict(h_dtype=3), {}), ("NULL rstd", dict(rstd=None), {}), ("d_residual: rows", dict(d_residual=9 << 20), {}),
    ("overlaps d_y", {}, dict(d_x=1 << 20)), ("overlaps h", {}, dict(d_x=(2 << 20) + 400)), ("d_x: NULL", {}, dict(d_x=None)),
    ("overlaps d_y", {}, dict(d_x2=(1 << 20) + 4)), ("-1 rows", dict(rows=-1), {}),
])
def test_norm_gradients_are_checked(needle, kw, more):
    lib = _lib().load()
    o = _norm_grad(**kw)
    _refused(lib.eg_add_rms_norm_grad(ctypes.byref(o), more.get("d_x", 6 << 20), 0, 300, more.get("d_x2"), 0, 300, None, None, 0, None), needle)


def test_norm_gradients_workspace():
    lib = _lib().load()
    size = lib.eg_add_rms_norm_grad_workspace_size
    assert size(5, 300) > 0 and size(0, 300) == 0 and size(-1, 300) == -1 and size(5, 20_481) == -1
    o = _norm_grad()
    args = (ctypes.byref(o), 6 << 20, 0, 300, None, 0, 0, 7 << 20)
    _refused(lib.eg_add_rms_norm_grad(*args, 8 << 20, size(5, 300) - 1, None), "workspace", _lib().EG_ERR_WORKSPACE)
    _refused(lib.eg_add_rms_norm_grad(*args, None, size(5, 300), None), "aligned")
    o = _norm_grad(d=20_481, dy_stride=20_481, h_stride=20_481)
    _refused(lib.eg_add_rms_norm_grad(ctypes.byref(o), 6 << 20, 0, 20_481, None, 0, 0, None, None, 0, None), "at most 20480", _lib().EG_ERR_UNSUPPORTED)


def _clip(*tensors, max_norm=1.0, norm=4096, ws=4096, n=1 << 30):
    lib = _lib()
    t = (lib.EgClipTensor * max(1, len(tensors)))()
    for to, (g, out, rows, cols, stride) in zip(t, tensors):
        to.g, to.out, to.rows, to.cols, to.g_stride, to.out_stride = g, out, rows, cols, stride, stride
    return lib.load().eg_clip_grads(t, len(tensors), max_norm, norm, ws, n, None)


def test_clipping_is_checked():
    a = (1 << 20, 1 << 20, 4, 100, 100)
    _refused(_clip(a, norm=None), "NULL norm")
    _refused(_clip(a, max_norm=-1.0), "max_norm")
    _refused(_clip(a, max_norm=float("nan")), "max_norm")
    _refused(_clip(a, ws=None), "aligned")
    _refused(_clip(a, n=0), "workspace", _lib().EG_ERR_WORKSPACE)
    _refused(_clip((None, None, 4, 100, 100)), "NULL")
    _refused(_clip((1 << 20, 1 << 20, 4, 100, 99)), "apart")
    _refused(_clip((1 << 20, 1 << 20, -1, 100, 100)), "is -1 x 100")
    _refused(_clip(a, a), "overlaps")
    _refused(_clip(a, ((1 << 20) + 1596, (1 << 20) + 1596, 4, 100, 100)), "overlaps")
    _refused(_clip((1 << 20, (1 << 20) + 4, 4, 100, 100)), "not in its place")
    _refused(_clip(a, (2 << 20, None, 4, 100, 100)), "some none")
    _refused(_clip((1 << 20, 3 << 20, 4, 100, 100), (3 << 20, 4 << 20, 4, 100, 100)), "overlaps")


def test_host_tensors_and_wrong_types_are_refused():
    from engraft_ngram_amd import clip, fp8, norm
    x = torch.zeros((3, 256))
    w = fp8.Fp8Weight(torch.zeros((5, 256), dtype=torch.uint8).view(torch.float8_e4m3fn),
                      torch.zeros((1, 4), dtype=torch.uint8).view(torch.float8_e8m0fnu), 256)
    for call in (lambda: fp8.quantize_rows(x), lambda: fp8.quantize_weight(x), lambda: fp8.product(x, w), lambda: norm.add_rms_norm(x, x),
                 lambda: norm.rms_norm(x), lambda: clip.grad_norm([x]), lambda: clip.clip_grads([x], 1.0), lambda: w.dequantize(),
                 lambda: norm.normed_product(x, x, None, w)):
        with pytest.raises(ValueError, match="GPU|on "):
            call()
    for call, needle in ((lambda: fp8.product(x.double(), w), "float32, bfloat16 or float16"), (lambda: fp8.product(x, w, out_dtype=torch.int32), "out_dtype"),
                         (lambda: fp8.product_grad(x, w), "transpose"), (lambda: fp8.product(x, w, split=-5), "split"),
                         (lambda: fp8.product(x.requires_grad_(), w), "transpose"), (lambda: clip.clip_grads([], 1.0), "no gradients"),
                         (lambda: clip.clip_grads([x], float("nan")), "max_norm"), (lambda: norm.add_rms_norm(x, x[:2]), "residual must be"),
                         (lambda: norm.rms_norm(torch.zeros(())), "rows"), (lambda: norm.normed_product(x[:, :5], None, None, w), "256 columns")):
        with pytest.raises(ValueError, match=needle):
            call()
