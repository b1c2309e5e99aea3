"""Memory that the 8-bit products write and must not share with what they read or write besides, refused on the host and before
any launch."""
from __future__ import annotations

import pytest

from tests.test_fp8_arguments import _lib, _matrix, _ref, _refused

MB = 1 << 20


def _rows(at, rows=5, k=300, **kw):
    return _matrix(rows, k, q=at, scales=at + MB // 2, **kw)


def _weight(at, rows=7, k=300):
    return _matrix(rows, k, 128, q=at, scales=at + MB // 2)


@pytest.mark.parametrize("x", [1 * MB, 1 * MB + 1900, MB + MB // 2, MB + MB // 2 - 5996, MB + MB // 2 + 16])
def test_blocks_of_rows(x):
    """Values in the place of the blocks or of their scales (5 x 300 values of 4 bytes; 5 x 384 bytes, 5 x 4 scales)."""
    _refused(_lib().load().eg_fp8_quantize(x, 0, 300, _ref(_rows(MB)), None), "overlap")


def test_blocks_on_their_own_scales():
    out = _rows(MB)
    out.scales = MB + 4 * 384
    _refused(_lib().load().eg_fp8_quantize(9 * MB, 0, 300, _ref(out), None), "overlap")


@pytest.mark.parametrize("x,col_stride,row_stride", [(MB, 1, 300), (MB + MB // 2, 1, 300), (2 * MB, 1, 300), (2 * MB + MB // 2 + 4, 1, 300), (MB, 7, 1),
                                                     (MB + 384 * 7 - 4, 1, 300)])
def test_blocks_of_weights(x, col_stride, row_stride):
    lib = _lib().load()
    w, t = _weight(MB), _weight(2 * MB, 300, 7)
    _refused(lib.eg_fp8_quantize_weight(x, 0, row_stride, col_stride, _ref(w), _ref(t), None), "overlap")


def test_blocks_of_weights_on_one_another():
    lib = _lib().load()
    w = _weight(MB)
    for t in (_weight(MB, 300, 7), _weight(MB + 128, 300, 7), _matrix(300, 7, 128, q=2 * MB, scales=MB + MB // 2),
              _matrix(300, 7, 128, q=2 * MB, scales=2 * MB + 128), _matrix(300, 7, 128, q=2 * MB, scales=MB + 300)):
        _refused(lib.eg_fp8_quantize_weight(9 * MB, 0, 300, 1, _ref(w), _ref(t), None), "overlap")


@pytest.mark.parametrize("out", [MB, MB + MB // 2, MB + 4 * 384 + 296, MB + MB // 2 - 5999 // 4 * 4])
def test_values_of_blocks(out):
    _refused(_lib().load().eg_fp8_dequantize(_ref(_rows(MB)), out, 0, 300, None), "overlap")


# a product's operands, as addresses that its outputs and its workspace must stay clear of
INPUTS = {"a": MB, "a's scales": MB + MB // 2, "b": 2 * MB, "b's scales": 2 * MB + MB // 2, "b2": 3 * MB, "b2's scales": 3 * MB + MB // 2}


@pytest.mark.parametrize("at", list(INPUTS.values()), ids=list(INPUTS))
@pytest.mark.parametrize("where", ["c", "c2"])
def test_outputs_of_products(at, where):
    lib = _lib().load()
    outs = {"c": 5 * MB, "c2": 6 * MB, where: at}
    _refused(lib.eg_fp8_product(_ref(_rows(MB)), _ref(_weight(2 * MB)), _ref(_weight(3 * MB)), outs["c"], 7, outs["c2"], 7, 0, None, 0, None), "overlap")
    if at == MB or at >= 2 * MB:  # values in the place of a's blocks
        _refused(lib.eg_fp8_linear(MB, 0, 5, 300, _ref(_weight(2 * MB)), _ref(_weight(3 * MB)), outs["c"], 7, outs["c2"], 7, 0, None, 0, None), "overlap")


@pytest.mark.parametrize("c2,ld", [(5 * MB, 7), (5 * MB + 24, 14), (5 * MB + 4 * (4 * 7 + 6), 7)])
def test_outputs_on_one_another(c2, ld):
    """5 x 7 outputs each; rows that lie between one another's are apart (a stride of 14 and an offset of 7), one column less are not."""
    lib = _lib().load()
    _refused(lib.eg_fp8_product(_ref(_rows(MB)), _ref(_weight(2 * MB)), _ref(_weight(3 * MB)), 5 * MB, ld, c2, ld, 0, None, 0, None), "overlap")


@pytest.mark.parametrize("ws", [4 * MB, 6 * MB, 6 * MB + MB // 2, 7 * MB, 8 * MB])
def test_the_workspace_of_products(ws):
    """100 x 10,240 values, in pieces: their sums and the rows' blocks are in the workspace."""
    lib = _lib().load()
    k, m = 10_240, 100
    need = lib.eg_fp8_product_workspace_size(m, 7, 9, k)
    a = _matrix(m, k, q=4 * MB, scales=5 * MB)  # (1,024,000 and 8,000 bytes)
    b, b2 = _matrix(7, k, 128, q=6 * MB, scales=6 * MB + MB // 2), _matrix(9, k, 128, q=9 * MB, scales=9 * MB + MB // 2)
    _refused(lib.eg_fp8_product(_ref(a), _ref(b), _ref(b2), 7 * MB, 7, 8 * MB, 9, 0, ws, need, None), "overlap")
    need = lib.eg_fp8_linear_workspace_size(m, 7, 9, k)
    x = MB  # 100 x 10,240 of 4 bytes: up to 4.9 MB
    _refused(lib.eg_fp8_linear(x, 0, m, k, _ref(b), _ref(b2), 7 * MB, 7, 8 * MB, 9, 0, ws, need, None), "overlap")
