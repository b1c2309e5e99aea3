"""The norm at the ends of the numbers' range, and its bounds as the kernels add today, on the GPU."""
from __future__ import annotations

import pytest
import torch

from tests import fp8_util as O
from tests.test_gpu_fp8 import HALF, SMALL
from tests.test_gpu_norm import _gen, _reference, _values

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = 2.0 ** -24
# eight squares in 32 bits: their own rounding and three additions, all terms positive; their sums and the root in 64, which halves
# it; the root's rounding to 32 (0.1: squares that are subnormal numbers, and the 64-bit steps)
ROOT = (4 / 2 + 1 + 0.1) * UNIT
NORM = ROOT + 2 * UNIT  # times the value and the weight


def _check(y, rstd, want, r, out):
    """``y`` and ``rstd`` against 64 bits; a root that is no normal fp32 number is the nearest one that there is."""
    fits = r[:, 0] <= torch.finfo(F32).max
    assert bool(rstd[~fits].isinf().all())
    off = (rstd.double() - r[:, 0]).abs()[fits]
    assert bool((off <= ROOT * r[:, 0][fits] + 2.0 ** -150).all()), float((off / r[:, 0][fits]).max() / UNIT)
    off = (y.double() - want).abs()
    bound = want.abs() * (NORM + (0.0 if out == F32 else HALF[out] * 1.001)) + SMALL[out]
    assert bool((off <= bound).all()), float((off / (want.abs() + 1e-300)).max() / UNIT)


@pytest.mark.parametrize("n,d", [(300, 1), (300, 7), (300, 128), (300, 600), (2000, 2560), (300, 2561), (300, 8192), (1000, 16_384),
                                 (100, 20_479)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
def test_the_root_is_of_64_bit_sums(cuda, n, d, dtype, out):
    from engraft_ngram_amd import norm
    g = _gen(n + d)
    x, w = _values(g, n, d, dtype), torch.randn(d, generator=g, device="cuda")
    _, _, r, want = _reference(x, None, w, 1e-5)
    y, _, rstd = norm.add_rms_norm_stats(x, None, w, eps=1e-5, out_dtype=out)
    _check(y, rstd, want, r, out)


# rows of these sizes: squares past the largest fp32 number and below the smallest, roots that are subnormal, and, of the last,
# larger than any
SIZES = [1e20, 1e38, 1e-22, 1e-30, 3e-38, 1e-41]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("d", [1, 7, 130, 600, 1000, 2560, 9001])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, "fp8")])
def test_squares_that_leave_32_bits(cuda, size, d, dtype, out):
    """Every third row is of ordinary size, and has the bits that it has alone."""
    from engraft_ngram_amd import norm
    n = 21
    g = _gen(d)
    x, w = torch.randn((n, d), generator=g, device="cuda"), torch.randn(d, generator=g, device="cuda")
    ordinary = torch.arange(n, device="cuda") % 3 == 1
    x = x.clamp_(-3.0, 3.0)
    x = torch.where(ordinary[:, None], x, x * size).to(dtype)
    x = torch.where((x == 0).all(1, keepdim=True), torch.tensor(max(size, 1e-40), dtype=dtype, device="cuda"), x)  # (a row of zeros is 0 / 0)
    _, _, r, want = _reference(x, None, w, 0.0)
    if out == "fp8":
        y = norm.rms_norm(x, w, eps=0.0, out_dtype="fp8")
        values, bytes_ = O.rows(want)
        near = (want * (1 - NORM), want * (1 + NORM))
        s = y.scales.view(torch.uint8).long()[:, :bytes_.shape[1]]
        assert bool(((s >= O.rows(near[0])[1]) & (s <= O.rows(near[1])[1])).all())
        scale = torch.exp2((s - 127).double()).repeat_interleave(128, 1)[:, :d]
        assert bool(((y.dequantize(F32).double() - want).abs() <= want.abs() * (2.0 ** -4 + NORM) + scale * 2.0 ** -10).all())
        alone = norm.rms_norm(x[ordinary], w, eps=0.0, out_dtype="fp8")
        assert torch.equal(y.q.view(torch.uint8)[ordinary], alone.q.view(torch.uint8))
        return
    y, _, rstd = norm.add_rms_norm_stats(x, None, w, eps=0.0, out_dtype=out)
    _check(y, rstd, want, r, out)
    alone = norm.add_rms_norm_stats(x[ordinary], None, w, eps=0.0, out_dtype=out)
    assert torch.equal(y[ordinary], alone[0]) and torch.equal(rstd[ordinary], alone[2])


@pytest.mark.parametrize("size", [1e20, 1e37, 1e-22, 1e-30])
def test_gradients_of_rows_whose_squares_leave_32_bits(cuda, size):
    """x, the residual and the weight through the sum of two such tensors."""
    from engraft_ngram_amd import norm
    g = _gen(5)
    x, res = (torch.randn((9, 700), generator=g, device="cuda") * size).requires_grad_(), torch.randn((9, 700), generator=g, device="cuda") * size
    w, d_y = torch.randn(700, generator=g, device="cuda").requires_grad_(), torch.randn((9, 700), generator=g, device="cuda")
    y, h = norm.add_rms_norm(x, res, w, eps=0.0)
    d_x, d_w = torch.autograd.grad(y, (x, w), d_y)
    _, v, r, _ = _reference(x.detach(), res, w.detach(), 0.0)
    u, p = v * r, d_y.double() * w.detach().double()
    want = r * (p - u * (p * u).mean(1, keepdim=True))
    bound = r * (p.abs() + u.abs() * (p * u).abs().mean(1, keepdim=True))
    # eight terms a lane in order, six additions across lanes, two wavefronts; 1 / d and the mean; u twice (its root and a product), p;
    # a product, a difference and the root's product
    adds = (8 + 6 + 2) + 2 + 2 * 4.1 + 1 + (3 + 3.1)
    assert bool(((d_x.double() - want).abs() <= bound * adds * UNIT + 2.0 ** -149).all())
    terms = d_y.double() * u
    assert bool(((d_w.double() - terms.sum(0)).abs() <= terms.abs().sum(0) * (9 + 16 + 6) * UNIT).all())


def test_zeros_and_what_is_not_finite(cuda):
    """The definition's: 0 / 0 without eps, zeros with it, and infinities and NaN as before."""
    from engraft_ngram_amd import norm
    for d in (5, 600, 2560):
        x = torch.zeros((6, d), device="cuda")
        assert bool(norm.rms_norm(x, eps=0.0).isnan().all()) and not bool(norm.rms_norm(x, eps=1e-30).any())
        x += 2.0
        x[2, 1], x[4, 0] = float("inf"), float("nan")
        y = norm.rms_norm(x, eps=0.0)
        assert bool((y[[0, 1, 3, 5]] == 1.0).all()) and bool(y[4].isnan().all())
        assert bool(y[2, 1].isnan()) and not bool(y[2, 2:].any()) and not bool(y[2, 0].any())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_eight_bits_round_as_the_exact_rows_do(cuda, dtype):
    """20 million values against the definition in 64 bits.  The roundings of the lanes' squares leave the root 2e-9 off (2^-24 of
    each of 320 sums, independent of each other), and a twelfth of a value lies between two borders: 0.4 values are expected to be on
    the other side, and 10 if the norm were in 32 bits."""
    from engraft_ngram_amd import norm
    g = _gen(77)
    w = torch.randn(2560, generator=g, device="cuda")
    others = 0
    for _ in range(8):
        x = _values(g, 1000, 2560, dtype)
        y = norm.rms_norm(x, w, eps=1e-6, out_dtype="fp8")
        want, bytes_ = O.rows(_reference(x, None, w, 1e-6)[3])
        assert int((y.scales.view(torch.uint8).long()[:, :20] != bytes_).sum()) <= 1
        others += int((y.dequantize(F32).double() != want).sum())
    assert others <= 3


@pytest.mark.parametrize("n,d", [(1, 64), (500, 130), (4100, 130), (1500, 2560), (700, 9000), (3000, 20_480)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_weights_gradient_as_it_is_added(cuda, n, d, dtype):
    from engraft_ngram_amd import norm
    g = _gen(n + d)
    h, d_y = _values(g, n, d, dtype), _values(g, n, d, dtype, 0.1)
    w = torch.randn(d, generator=g, device="cuda")
    _, _, rstd = norm.add_rms_norm_stats(h, None, w, eps=1e-5)
    _, d_w = norm.add_rms_norm_grad(d_y, h, rstd, w)
    _, v, r, _ = _reference(h, None, w, 1e-5)
    terms = d_y.double() * v * r
    pieces = -(-d // 512)
    held = -(-pieces // 16)
    wavefronts = -(-pieces // held)
    at_once = max(1, 16 // wavefronts)  # rows of a workgroup
    groups = min(-(-n // at_once), 512)
    adds = -(-n // (groups * at_once)) + at_once + -(-groups // 16) + 16
    assert bool(((d_w.double() - terms.sum(0)).abs() <= terms.abs().sum(0) * (adds * UNIT + ROOT + 2 * UNIT) + 2.0 ** -126).all())
