"""Operands and outputs of the 8-bit products in one buffer, apart but between one another's rows, on the GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_gpu_fp8 import _gen, _values

pytestmark = pytest.mark.gpu


def _matrix(q, scales, k, rows, block_rows):
    from engraft_ngram_amd import _lib
    return _lib.EgFp8Matrix(q.data_ptr(), scales.data_ptr(), rows, k, q.stride(0), scales.stride(0), block_rows)


@pytest.mark.parametrize("m,k,n,n2", [(3, 300, 200, 72), (40, 300, 200, 72), (100, 10_240, 72, 200), (2047, 640, 256, 128)])
def test_outputs_and_values_side_by_side(cuda, m, k, n, n2):
    """Rows of x, then of both outputs: the strides that a caller's one buffer of rows has."""
    from engraft_ngram_amd import _lib, fp8
    g = _gen(m)
    w, w2 = (fp8.quantize_weight(_values(g, rows, k, torch.float32, 0.02), transpose=False) for rows in (n, n2))
    buffer = torch.full((m, k + n + n2), float("nan"), device="cuda")
    buffer[:, :k] = _values(g, m, k, torch.float32)
    x, c, c2 = buffer[:, :k], buffer[:, k:k + n], buffer[:, k + n:]
    ld = buffer.stride(0)
    b, b2 = _matrix(w.q, w.scales, k, n, 128), _matrix(w2.q, w2.scales, k, n2, 128)
    need = _lib.load().eg_fp8_linear_workspace_size(m, n, n2, k)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    kept = x.clone()
    _lib.call("eg_fp8_linear", x.data_ptr(), 0, m, ld, ctypes.byref(b), ctypes.byref(b2), c.data_ptr(), ld, c2.data_ptr(), ld, 0,
              ws.data_ptr() if need else None, need, _lib.stream_ptr())
    assert torch.equal(x, kept)
    for got, weight in ((c, w), (c2, w2)):
        want = fp8.product(kept, weight)
        assert float((got - want).norm()) <= 1e-5 * float(want.norm())  # (the order of a sum goes by both outputs' sizes)


def test_blocks_and_values_side_by_side(cuda):
    """Each row's values, its blocks and its scales one behind the other."""
    from engraft_ngram_amd import _lib, fp8
    m, k = 50, 300
    x = _values(_gen(1), m, k, torch.bfloat16)
    row = 608 + 384 + 16  # bytes: 300 values and a gap, three blocks, three scales and their fill
    buffer = torch.zeros((m, row), dtype=torch.uint8, device="cuda")
    buffer[:, :600] = x.view(torch.uint8)
    out = _lib.EgFp8Matrix(buffer.data_ptr() + 608, buffer.data_ptr() + 992, m, k, row, row, 1)
    _lib.call("eg_fp8_quantize", buffer.data_ptr(), 1, row // 2, ctypes.byref(out), _lib.stream_ptr())
    want = fp8.quantize_rows(x)
    assert torch.equal(buffer[:, 608:992], want.q.view(torch.uint8)) and torch.equal(buffer[:, 992:996], want.scales.view(torch.uint8))
    assert torch.equal(buffer[:, :600], x.view(torch.uint8))
    _lib.call("eg_fp8_dequantize", ctypes.byref(out), buffer.data_ptr(), 1, row // 2, _lib.stream_ptr())
    assert torch.equal(buffer[:, :600].contiguous().view(torch.bfloat16), want.dequantize())
