"""Products of 8-bit blocks in every tile that the sizes can choose, at every type of output, and at the ends of the scales'
range."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_gpu_fp8 import BF16, F16, F32, HALF, SMALL, _gen, _values, check_product

# m, k, n, split: ragged rows, columns and blocks; one and two groups of columns, which may end inside a tile
SIZES = [(1, 700, 300, None), (20, 700, 300, 128), (777, 1000, 1111, None), (777, 1000, 1111, 640), (76, 5100, 125, None), (90, 5100, 700, 384),
         (1000, 640, 3100, None), (327, 300, 8194, 2560), (900, 1280, 8000, None), (1500, 300, 4100, 1152), (1161, 300, 6936, None),
         (2000, 640, 5000, 2432), (1287, 300, 8207, None), (1800, 300, 6950, 128), (3000, 640, 4100, 2560), (3000, 640, 6300, None),
         (1936, 300, 8209, None), (3000, 640, 6300, 2432), (2047, 2560, 10_240, None), (2047, 2560, 2560, None), (1921, 2433, 2400, 1280),
         (1024, 5248, 2560, None), (1000, 5100, 2500, 640), (16_376, 300, 1300, None)]
TILES = {(64, 64), (64, 128), (64, 160), (128, 128), (128, 160), (256, 192), (256, 256), (256, 320)}


def _plan(m, k, n, split, code):
    """((rows, columns) of the tile, pieces of k)"""
    from engraft_ngram_amd import _lib
    pieces = ctypes.c_int32()
    tile = _lib.load().eg_fp8_product_tile(m, split or n, n - split if split else 0, k, code, ctypes.byref(pieces))
    return (tile >> 16, tile & 0xFFFF), pieces.value


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("groups", [1, 2])
def test_the_sizes_take_every_tile(code, groups):
    """A tile that no size here chooses any more would go untested: then sizes have to be added."""
    plans = {_plan(*size, code) for size in SIZES}
    assert {tile for tile, pieces in plans if pieces == 1} == TILES | {(0, 0)}
    assert any(pieces > 1 for _, pieces in plans)
    # two groups of columns: in the tiles with an uneven share of loads, the kernel of few rows, and in pieces
    plans = {_plan(*size, code) for size in SIZES if (size[3] is not None) == (groups == 2)}
    assert {(0, 0), (64, 64), (64, 160), (128, 160), (256, 320)} <= {tile for tile, _ in plans} and any(p > 1 for _, p in plans)


def test_plans_out_of_range():
    from engraft_ngram_amd import _lib
    tile = _lib.load().eg_fp8_product_tile
    assert tile(-1, 5, 0, 300, 0, None) == -1 and tile(5, 5, 0, 0, 0, None) == -1 and tile(5, 5, 0, 300, 3, None) == -1
    assert tile(500, 0, 0, 300, 0, None) == 0 and tile(0, 5, 0, 300, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,split", SIZES)
@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_tiles(cuda, m, k, n, split, out):
    """Against 64 bits; rows and columns behind the outputs stay as they are."""
    from engraft_ngram_amd import _lib, fp8
    g = _gen(m + k + n)
    x, w = fp8.quantize_rows(_values(g, m, k, BF16)), fp8.quantize_weight(_values(g, n, k, F32, 0.02), transpose=False)
    parts = fp8.product(x, w, out_dtype=out, split=split)
    parts = parts if split else (parts,)
    check_product(torch.cat(parts, 1), x.dequantize(F32).double(), w.dequantize().double(), out, out == F32)

    def matrix(q, scales, rows, block_rows):
        return _lib.EgFp8Matrix(q.data_ptr(), scales.data_ptr(), rows, k, q.stride(0), scales.stride(0), block_rows)

    first = split or n
    a, b = matrix(x.q, x.scales, m, 1), matrix(w.q, w.scales, first, 128)
    b2 = matrix(w.q[first:], w.scales[first // 128:], n - first, 128) if split else None
    buffers = [torch.full((m + 3, part.shape[1] + 5), float("nan"), dtype=out, device="cuda") for part in parts]
    code = _lib.dtype_code(out)
    need = _lib.load().eg_fp8_product_workspace_size(m, first, n - first, k)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    c = [(t[1:, 2:].data_ptr(), t.stride(0)) for t in buffers] + [(None, 0)]
    _lib.call("eg_fp8_product", ctypes.byref(a), ctypes.byref(b), ctypes.byref(b2) if split else None, *c[0], *c[1], code, ws.data_ptr(), need,
              _lib.stream_ptr())
    for t, part in zip(buffers, parts):
        inside = t[1:m + 1, 2:part.shape[1] + 2]
        assert torch.equal(inside, part)
        inside.fill_(float("nan"))
        assert bool(t.isnan().all())


def _blocks(g, rows, k, bytes_, block_rows):
    """e4m3 values up to 240 under scales of these bytes, and what they stand for."""
    kp = -(-k // 128) * 128
    q = torch.randint(0, 120, (rows, kp), generator=g, device="cuda") + 128 * torch.randint(0, 2, (rows, kp), generator=g, device="cuda")
    q[:, k:] = 0
    scales = bytes_[torch.randint(0, len(bytes_), (-(-rows // block_rows), -(-kp // 512) * 4), generator=g, device="cuda")]
    scale = torch.exp2(scales.double() - 127).repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    q = q.to(torch.uint8).view(torch.float8_e4m3fn)
    return q, scales.to(torch.uint8).view(torch.float8_e8m0fnu), q[:, :k].float().double() * scale


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", [((0,), (127,)), ((0,), (227,)), ((127,), (0,)), ((227,), (0,)), ((1, 2), (200,)), ((3, 4), (200,)), ((247,), (7,)),
                                 ((247,), (0,)), ((7,), (247,)), ((240,), (10, 0)), ((0, 3, 120, 127), (0, 127, 130, 240))])
@pytest.mark.parametrize("m,k,n", [(1, 300, 200), (20, 2560, 200), (40, 300, 200), (2047, 640, 2560)])
@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_the_ends_of_the_scales(cuda, a, b, m, k, n, out):
    """Scales from 2^-127 to 2^120, which blocks can have.  f32 outputs take the values as bf16: those below 2^-126, which scales below
    2^-124 give, are rounded to its subnormal numbers, by up to 2^-134."""
    from engraft_ngram_amd import fp8
    g = _gen(m + n + k)
    bytes_ = [torch.tensor(x, device="cuda") for x in (a, b)]
    (xq, xs, xv), (wq, ws, wv) = _blocks(g, m, k, bytes_[0], 1), _blocks(g, n, k, bytes_[1], 128)
    y = fp8.product(fp8.Fp8Rows(xq, xs, k), fp8.Fp8Weight(wq, ws, k), out_dtype=out).double()
    want, size = xv @ wv.T, xv.abs() @ wv.abs().T
    slack = size * (k + 8) * 2.0 ** -24
    if out == F32:
        for v, other in ((xv, wv), (wv, xv)):
            lost = (v.abs() < 2.0 ** -126).double() * 2.0 ** -134 @ other.abs().T
            slack = slack + (lost if v is xv else lost.T)
    else:
        slack = slack + size * 2.0 ** -10
    off = (y - want).abs()
    largest = torch.finfo(out).max
    sums = size < torch.finfo(F32).max / 2  # (infinities of both signs meet in those past it)
    fits = sums & (want.abs() + slack < largest)
    bound = slack + (want.abs() + slack) * HALF[out] * 1.001 + SMALL[out]
    assert bool((off <= bound)[fits].all()), float((off / (size + 1e-300))[fits].max())
    past = sums & (want.abs() - slack > largest * (1 + HALF[out]))
    assert bool((y[past].abs() >= largest).all()) and bool((y[past].sign() == want[past].sign()).all())
