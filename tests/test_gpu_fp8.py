"""Products of 8-bit blocks against their definition in 64 bits, on the GPU."""
from __future__ import annotations

import pytest
import torch

from tests import fp8_util as O

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}  # half a step, relative, of a rounding
SMALL = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -25}  # half a step of the subnormal numbers, or below it


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(g, m, k, dtype, scale=1.0):
    x = torch.randn((m, k), generator=g, device="cuda") * torch.exp(torch.randn((1, k), generator=g, device="cuda"))
    return (x * scale).to(dtype)


def check_product(y, xv, wv, dtype, exact):
    """``y`` against ``xv @ wv.T`` of float64 values: fp32 sums are off by at most k 2^-24 of the sum of magnitudes; the fp8
    matrix cores drop of each of eight products less than 2^-13 of the largest, 2^-10 of a group's magnitudes."""
    want = xv @ wv.T
    size = xv.abs() @ wv.abs().T
    slack = size * (xv.shape[1] + 8) * 2.0 ** -24 + (0.0 if exact else size * 2.0 ** -10)
    off = (y.double() - want).abs()
    assert bool((off <= slack + (want.abs() + slack) * HALF[dtype] * 1.001 + SMALL[dtype]).all()), float((off / (size + 1e-300)).max())
    # as a whole: rounding errors do not add up to their bounds (fp32 sums 1e-7 of the result, dropped parts 1.5e-5)
    norm = float(want.norm())
    if norm > 0 and want.numel() > 64:
        assert float(off.norm()) <= norm * (1e-6 + (0.0 if exact else 1e-4) + HALF[dtype])


# ---- blocks ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 640), (7, 1000), (300, 2560)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_are_the_definitions(cuda, m, k, dtype):
    from engraft_ngram_amd import fp8
    x = _values(_gen(m * 1000 + k), m, k, dtype)
    if m > 1:
        x[1] = 0.0
        x[0, 0] = float("nan")
        x[0, -1] = float("inf")
    r = fp8.quantize_rows(x)
    want, bytes_ = O.rows(x)
    nb = bytes_.shape[1]
    s = r.scales.view(torch.uint8).long()
    assert torch.equal(s[:, :nb], bytes_) and bool((s[:, nb:] == 127).all())
    assert bool((r.q.view(torch.uint8)[:, k:] == 0).all())
    for t in (F32, BF16):
        assert torch.equal(torch.nan_to_num(r.dequantize(t).double(), nan=1e9), torch.nan_to_num(want, nan=1e9))


def test_rows_at_the_edges_of_a_scale(cuda):
    """448 2^e and its neighbours, the smallest and largest numbers, subnormal ones."""
    from engraft_ngram_amd import fp8
    tops = []
    for e in (-140, -127, -100, -9, 0, 1, 100, 119):
        t = torch.tensor(448.0 * 2.0 ** e if e > -140 else 2.0 ** -140, dtype=F32)
        tops += [t, torch.nextafter(t, t * 2), torch.nextafter(t, t * 0)]
    tops += [torch.tensor(torch.finfo(F32).max), torch.tensor(2.0 ** -149)]
    x = torch.zeros((len(tops), 130))
    for i, t in enumerate(tops):
        x[i, 5], x[i, 6], x[i, 129] = t, -t / 3, t / 7
    x = x.cuda()
    r = fp8.quantize_rows(x)
    want, bytes_ = O.rows(x)
    assert torch.equal(r.scales.view(torch.uint8).long()[:, :2], bytes_)
    got = r.dequantize(F32).double()
    normal = want.abs() >= 2.0 ** -126
    # the largest fp32 number, (2 - 2^-23) 2^127, becomes 16 steps of 2^124: 2^128, which is no fp32 number
    assert torch.equal(got[normal], want[normal].float().double())
    assert bool(((got - want).abs()[~normal] <= 2.0 ** -126).all())


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (300, 1000), (1111, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_and_their_transposes(cuda, n, k, dtype):
    from engraft_ngram_amd import fp8
    w = _values(_gen(n + k), n, k, dtype, 0.02)
    wide = torch.empty((n, k + 5), dtype=dtype, device="cuda")
    wide[:, 3:k + 3] = w
    for view in (w, w.T.contiguous().T, wide[:, 3:k + 3]):
        q = fp8.quantize_weight(view)
        want, bytes_ = O.rows(w, 128)
        assert q.shape == (n, k)
        assert torch.equal(q.dequantize().double(), want)
        assert torch.equal(q.scales.view(torch.uint8).long()[:, :bytes_.shape[1]], bytes_)
        assert bool((q.scales.view(torch.uint8)[:, bytes_.shape[1]:] == 127).all())
        t = fp8.Fp8Weight(q.q_t, q.scales_t, n)
        assert torch.equal(t.dequantize().double(), want.T)
        assert bool((q.q.view(torch.uint8)[:, k:] == 0).all()) and bool((q.q_t.view(torch.uint8)[:, n:] == 0).all())
        assert bool((q.scales_t.view(torch.uint8)[:, bytes_.shape[0]:] == 127).all())
        alone = fp8.quantize_weight(view, transpose=False)
        assert alone.q_t is None and torch.equal(alone.q.view(torch.uint8), q.q.view(torch.uint8))


# ---- products --------------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 2560, 640), (2, 130, 17), (4, 700, 300), (5, 128, 129), (16, 2560, 272), (17, 1000, 500), (32, 256, 128),
         (33, 640, 200), (64, 2560, 64), (65, 129, 257), (127, 1000, 1111), (300, 384, 2048), (777, 1000, 1111), (1500, 640, 4100),
         (2047, 2560, 4100), (70, 5000, 130), (200, 10_240, 2560), (65, 4096, 1)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)])
def test_products(cuda, m, k, n, dtype, out):
    from engraft_ngram_amd import fp8
    g = _gen(m + k + n)
    x, w = _values(g, m, k, dtype), fp8.quantize_weight(_values(g, n, k, F32, 0.02), transpose=False)
    y = fp8.product(x, w, out_dtype=out)
    assert y.shape == (m, n) and y.dtype == out
    xv, wv = O.rows(x)[0], w.dequantize().double()
    exact = out == F32
    check_product(y, xv, wv, out, exact)
    # the same from blocks, and the same bits again
    r = fp8.quantize_rows(x)
    assert torch.equal(fp8.product(r, w, out_dtype=out), y) or m <= 32  # few rows take their own blocks in a kernel of its own order
    check_product(fp8.product(r, w, out_dtype=out), xv, wv, out, exact)
    assert torch.equal(fp8.product(x, w, out_dtype=out), y)


@pytest.mark.parametrize("m,k,n,split", [(2047, 2560, 2560, None), (1900, 2300, 2501, None), (1921, 2433, 2400, 1280),
                                         (1024, 5248, 2560, None), (1000, 5100, 2500, 640)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_products_of_long_rows(cuda, m, k, n, split, out):
    """As many tiles as CUs, whose wavefronts take halves of the blocks: whole and ragged, an even and an odd number of blocks."""
    from engraft_ngram_amd import fp8
    g = _gen(m + k)
    x, w = _values(g, m, k, BF16), fp8.quantize_weight(_values(g, n, k, F32, 0.02), transpose=False)
    y = fp8.product(x, w, out_dtype=out, split=split)
    y = torch.cat(y, 1) if split else y
    check_product(y, O.rows(x)[0], w.dequantize().double(), out, out == F32)
    again = fp8.product(x, w, out_dtype=out, split=split)
    assert torch.equal(torch.cat(again, 1) if split else again, y)


@pytest.mark.parametrize("m,k,n", [(1, 640, 200), (24, 1000, 300), (130, 300, 700), (600, 2560, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient(cuda, m, k, n, dtype):
    from engraft_ngram_amd import fp8
    g = _gen(m)
    w = fp8.quantize_weight(_values(g, n, k, F32, 0.02))
    x = _values(g, m, k, dtype).requires_grad_()
    d_y = _values(g, m, n, dtype, 1e-2)
    y = fp8.product(x, w)
    (d_x,) = torch.autograd.grad(y, x, d_y)
    assert d_x.shape == x.shape and d_x.dtype == dtype
    check_product(d_x, O.rows(d_y)[0], w.dequantize().double().T.contiguous(), dtype, dtype == F32)
    assert torch.equal(fp8.product_grad(d_y, w), d_x)


def test_split_leads_and_strides(cuda):
    """Two outputs, leading dimensions, rows of a wider buffer, a transposed x, rows expanded from one."""
    from engraft_ngram_amd import fp8
    g = _gen(3)
    w = fp8.quantize_weight(_values(g, 300, 260, F32, 0.02))
    for m in (3, 20, 40):
        x = _values(g, 2 * m, 260, BF16)
        whole = fp8.product(x, w, out_dtype=F32)
        a, b = fp8.product(x, w, out_dtype=F32, split=128)
        assert torch.equal(torch.cat([a, b], 1), whole) and a.is_contiguous() and b.is_contiguous()
        assert torch.equal(fp8.product(x.reshape(2, m, 260), w, out_dtype=F32), whole.reshape(2, m, 300))
        wide = torch.full((2 * m, 267), float("nan"), dtype=BF16, device="cuda")
        wide[:, 5:265] = x
        assert torch.equal(fp8.product(wide[:, 5:265], w, out_dtype=F32), whole)
        assert torch.equal(fp8.product(x.T.contiguous().T, w, out_dtype=F32), whole)
        one = x[:1].expand(m, 260)
        assert torch.equal(fp8.product(one, w, out_dtype=F32), fp8.product(one.contiguous(), w, out_dtype=F32))
        leaf = x.float().requires_grad_()
        a, b = fp8.product(leaf, w, split=128)
        (one_grad,) = torch.autograd.grad(b.sum(), leaf)
        d = torch.zeros((2 * m, 300), device="cuda")
        d[:, 128:] = 1.0
        assert torch.equal(one_grad, fp8.product_grad(d, w))
    assert fp8.product(x[:0], w).shape == (0, 300)


def test_what_is_not_finite_stays_in_its_rows_and_columns(cuda):
    from engraft_ngram_amd import fp8
    g = _gen(4)
    for m in (3, 20, 70, 400):
        x, wf = _values(g, m, 300, F32), _values(g, 200, 300, F32, 0.02)
        x[1, 7], x[2, 299], wf[9, 5] = float("inf"), float("nan"), float("nan")
        w = fp8.quantize_weight(wf)
        for out in (F32, BF16):
            y = fp8.product(x, w, out_dtype=out)
            bad = torch.zeros((m, 200), dtype=torch.bool, device="cuda")
            bad[1] = bad[2] = True
            bad[:, 9] = True
            assert torch.equal(y.isnan(), bad)


def test_rows_of_views_and_rows_behind(cuda):
    """Blocks of some rows of a larger matrix: what lies behind them is neither read nor has a part."""
    from engraft_ngram_amd import fp8
    g = _gen(5)
    x, w = _values(g, 90, 384, BF16), fp8.quantize_weight(_values(g, 100, 384, F32, 0.02))
    r = fp8.quantize_rows(x)
    for last in (12, 50, 89):
        want = fp8.product(fp8.quantize_rows(x[10:last].contiguous()), w)
        r.q.view(torch.uint8)[last:] = 0x7F  # NaN
        r.scales.view(torch.uint8)[last:] = 0xFF
        part = fp8.Fp8Rows(r.q[10:last], r.scales[10:last], 384)
        assert torch.equal(fp8.product(part, w), want)
        r = fp8.quantize_rows(x)


def test_streams_and_graphs(cuda):
    """On another stream than the tensors', and captured: replays see new inputs and agree with eager calls."""
    from engraft_ngram_amd import fp8
    g = _gen(6)
    w = fp8.quantize_weight(_values(g, 500, 640, F32, 0.02))
    for m in (1, 20, 200):
        x = _values(g, m, 640, BF16)
        d = _values(g, m, 500, BF16)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y = fp8.product(x, w)
        side.synchronize()
        assert torch.equal(y, fp8.product(x, w))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, d_x = fp8.product(x, w), fp8.product_grad(d, w)
        for k in range(3):
            x.copy_(_values(g, m, 640, BF16))
            d.copy_(_values(g, m, 500, BF16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, fp8.product(x, w)) and torch.equal(d_x, fp8.product_grad(d, w)), (m, k)


def test_rows_past_4_gib(cuda):
    """Rows whose bytes lie more than 2^32 apart."""
    from engraft_ngram_amd import fp8
    m, k, n = 1_700_000, 2560, 8
    g = _gen(7)
    r = fp8.Fp8Rows(torch.zeros((m, k), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                    torch.full((m, 20), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu), k)
    some = fp8.quantize_rows(_values(g, 100, k, F32))
    w = fp8.quantize_weight(_values(g, n, k, F32, 0.02), transpose=False)
    r.q.view(torch.uint8)[-100:] = some.q.view(torch.uint8)
    r.scales.view(torch.uint8)[-100:] = some.scales.view(torch.uint8)
    y = fp8.product(r, w, out_dtype=F32)
    assert not bool(y[:-100].any())
    check_product(y[-100:], some.dequantize(F32).double(), w.dequantize().double(), F32, True)
    # and values and outputs more than 2^32 bytes apart
    x = torch.zeros((m, k), dtype=BF16, device="cuda")
    x[-100:] = _values(g, 100, k, BF16)
    last = fp8.quantize_rows(x[-100:])
    assert torch.equal(fp8.quantize_rows(x).q[-100:].view(torch.uint8), last.q.view(torch.uint8))
    w = fp8.quantize_weight(_values(g, 1300, k, F32, 0.02), transpose=False)
    y = fp8.product(x, w, out_dtype=BF16)
    assert not bool(y[:-100].any()) and torch.equal(y[-100:], fp8.product(x[-300:], w, out_dtype=BF16)[-100:])


def test_a_weight_that_changed_before_the_gradient(cuda):
    from engraft_ngram_amd import fp8
    g = _gen(8)
    w = fp8.quantize_weight(_values(g, 200, 300, F32, 0.02))
    y = fp8.product(_values(g, 50, 300, F32).requires_grad_(), w)
    w.q_t.view(torch.uint8).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_captured(cuda):
    """Forward and backward through autograd in one graph: replays see new inputs."""
    from engraft_ngram_amd import fp8, norm
    g = _gen(9)
    w = fp8.quantize_weight(_values(g, 300, 640, F32, 0.02))
    x, res, d = _values(g, 70, 640, BF16).requires_grad_(), _values(g, 70, 640, BF16), _values(g, 70, 300, BF16)
    nw = torch.randn(640, generator=g, device="cuda").requires_grad_()

    def step():
        y, h = norm.normed_product(x, res, nw, w)
        return (y.detach(), *torch.autograd.grad(y, (x, nw), d))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(_values(g, 70, 640, BF16))
            d.copy_(_values(g, 70, 300, BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
