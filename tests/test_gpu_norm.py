"""The residual's norm and its gradients against the formulas in 64 bits, on the GPU."""
from __future__ import annotations

import pytest
import torch

from tests import fp8_util as O
from tests.test_gpu_fp8 import HALF, SMALL

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# the sum of squares: at most 40 values a lane in order, 6 additions across lanes, 16 across wavefronts, half of
# that in its root; the root, the quotient and two products
NORM = (62 / 2 + 6) * 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(g, n, d, dtype, scale=1.0):
    return (torch.randn((n, d), generator=g, device="cuda") * torch.exp(torch.randn(d, generator=g, device="cuda")) * scale).to(dtype)


def _reference(x, residual, w, eps):
    h = x if residual is None else (x.double() + residual.double()).to(residual.dtype)
    # the addition is in fp32 before it is rounded
    if residual is not None:
        h = (x.float() + residual.float()).to(residual.dtype)
    v = h.double()
    r = 1.0 / torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + eps)
    return h, v, r, v * r * (1.0 if w is None else w.double())


WIDTHS = [(1, 1), (3, 7), (2, 128), (5, 511), (4, 513), (9, 2560), (1200, 2560), (3, 4097), (40, 16_384), (2, 20_480), (2100, 130), (3, 1023), (5, 2561), (700, 20_479)]


@pytest.mark.parametrize("n,d", WIDTHS)
@pytest.mark.parametrize("dtype,r_dtype,out", [(F32, F32, F32), (BF16, BF16, BF16), (F16, F16, F16), (BF16, F32, BF16), (F16, None, F32), (F32, None, BF16)])
def test_norms(cuda, n, d, dtype, r_dtype, out):
    from engraft_ngram_amd import norm
    g = _gen(n + d)
    x = _values(g, n, d, dtype)
    res = None if r_dtype is None else _values(g, n, d, r_dtype)
    w = torch.randn(d, generator=g, device="cuda").to(dtype) if d != 7 else None
    h_want, _, r, want = _reference(x, res, w, 1e-5)
    y, h, rstd = norm.add_rms_norm_stats(x, res, w, eps=1e-5, out_dtype=out)
    assert y.dtype == out and torch.equal(h, h_want)
    assert bool(((rstd.double() - r[:, 0]).abs() <= NORM * r[:, 0]).all())
    off = (y.double() - want).abs()
    assert bool((off <= want.abs() * (NORM + HALF[out] * 1.001) + SMALL[out]).all())
    if res is None:
        assert torch.equal(norm.rms_norm(x, w, eps=1e-5, out_dtype=out), y)
    else:
        again = norm.add_rms_norm(x, res, w, eps=1e-5, out_dtype=out)
        assert torch.equal(again[0], y) and torch.equal(again[1], h)


@pytest.mark.parametrize("n,d", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norms_in_blocks(cuda, n, d, dtype):
    """Each value is within half a step of e4m3 under its block's scale of the formula's, and each scale is the formula's but where
    the block's largest value is within the norm's error of the border."""
    from engraft_ngram_amd import norm
    g = _gen(n + d + 1)
    x, res = _values(g, n, d, dtype), _values(g, n, d, dtype)
    if n > 2:
        x[1], res[1] = 0.0, 0.0
    w = torch.randn(d, generator=g, device="cuda")
    h_want, _, _, want = _reference(x, res, w, 1e-5)
    y, h = norm.add_rms_norm(x, res, w, eps=1e-5, out_dtype="fp8")
    assert torch.equal(h, h_want) and y.shape == (n, d)
    nb = -(-d // 128)
    s = y.scales.view(torch.uint8).long()
    low, high = O.rows(want * (1 - NORM))[1], O.rows(want * (1 + NORM))[1]
    assert bool(((s[:, :nb] >= low) & (s[:, :nb] <= high)).all()) and bool((s[:, nb:] == 127).all())
    scale = torch.exp2((s[:, :nb] - 127).double()).repeat_interleave(128, 1)[:, :d]
    off = (y.dequantize(F32).double() - want).abs()
    assert bool((off <= want.abs() * (2.0 ** -4 + NORM * 1.1) + scale * 2.0 ** -10 + 2.0 ** -126).all())
    assert bool((y.q.view(torch.uint8)[:, d:] == 0).all())


@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (5, 511), (9, 2560), (1500, 2560), (3, 4097), (40, 16_384), (2, 20_480), (4100, 130), (0, 64), (1300, 2559), (300, 20_473)])
@pytest.mark.parametrize("dy_dtype,dtype", [(F32, F32), (BF16, BF16), (F32, F16), (BF16, F32)])
def test_gradients(cuda, n, d, dy_dtype, dtype):
    from engraft_ngram_amd import norm
    g = _gen(n * 3 + d)
    h, d_y = _values(g, n, d, dtype), _values(g, n, d, dy_dtype, 0.1)
    w = torch.randn(d, generator=g, device="cuda")
    d_res = _values(g, n, d, dtype, 0.1) if d != 511 else None
    _, _, rstd = norm.add_rms_norm_stats(h, None, w, eps=1e-5)
    d_h, d_w = norm.add_rms_norm_grad(d_y, h, rstd, w, d_residual=d_res, dtype=F32)
    _, v, r, _ = _reference(h, None, w, 1e-5)
    u, p = v * r, d_y.double() * w.double()
    base = 0.0 if d_res is None else d_res.double()
    want = base + r * (p - u * (p * u).mean(1, keepdim=True))
    # a row's sum as the norm's; its terms and the result a few roundings each
    size = (0.0 if d_res is None else d_res.double().abs()) + r * (p.abs() + u.abs() * (p * u).abs().mean(1, keepdim=True))
    assert bool(((d_h.double() - want).abs() <= size * (62 + 40 + 12) * 2.0 ** -24 + 2.0 ** -126).all())
    terms = d_y.double() * u
    # a wavefront's rows in order, the workgroup's, a quarter of the partial sums in order
    adds = n / 256 + 4 + 128 + 40
    assert bool(((d_w.double() - terms.sum(0)).abs() <= terms.abs().sum(0) * adds * 2.0 ** -24 + 2.0 ** -126).all())
    rounded, _ = norm.add_rms_norm_grad(d_y, h, rstd, w, d_residual=d_res)
    assert torch.equal(rounded, d_h.to(dtype))
    again = norm.add_rms_norm_grad(d_y, h, rstd, w, d_residual=d_res, dtype=F32)
    assert torch.equal(again[0], d_h) and torch.equal(again[1], d_w)


@pytest.mark.parametrize("dtype,r_dtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
def test_autograd(cuda, dtype, r_dtype):
    """All inputs' gradients through both outputs, through one of them, and with leading dimensions."""
    from engraft_ngram_amd import norm
    g = _gen(8)
    x = _values(g, 30, 300, dtype).reshape(5, 6, 300).requires_grad_()
    res = _values(g, 30, 300, r_dtype).reshape(5, 6, 300).requires_grad_()
    w = torch.randn(300, generator=g, device="cuda").requires_grad_()
    d_y, d_h = _values(g, 30, 300, dtype).reshape(5, 6, 300), _values(g, 30, 300, r_dtype).reshape(5, 6, 300)
    y, h = norm.add_rms_norm(x, res, w)
    assert y.shape == x.shape and h.dtype == r_dtype
    _, _, rstd = norm.add_rms_norm_stats(x.detach().reshape(30, 300), res.detach().reshape(30, 300), w.detach())
    for use_y, use_h in ((True, True), (True, False), (False, True)):
        outs = [o for o, use in ((y, use_y), (h, use_h)) if use]
        ds = [d for d, use in ((d_y, use_y), (d_h, use_h)) if use]
        gx, gr, gw = torch.autograd.grad(outs, (x, res, w), ds, retain_graph=True)
        assert gx.shape == x.shape and gx.dtype == dtype and gr.dtype == r_dtype
        if use_y:
            want, want_w = norm.add_rms_norm_grad(d_y.reshape(30, 300), h.detach().reshape(30, 300), rstd, w.detach(),
                                                  d_residual=d_h.reshape(30, 300) if use_h else None, dtype=F32)
            assert torch.equal(gw, want_w)
        else:
            want = d_h.reshape(30, 300).float()
            assert not bool(gw.any())
        assert torch.equal(gx.reshape(30, 300), want.to(dtype)) and torch.equal(gr.reshape(30, 300), want.to(r_dtype))
    only = torch.autograd.grad(y, w, d_y, retain_graph=True)[0]
    assert torch.equal(only, torch.autograd.grad(y, (w, x), d_y)[0])
    z = norm.rms_norm(x.detach().requires_grad_(), None)
    z.sum().backward()


def test_gradient_against_differences(cuda):
    """The autograd function's gradients of a random projection of both outputs against central differences of the formula in
    64 bits (a step of 1e-4 leaves 1e-7 of the third derivative)."""
    from engraft_ngram_amd import norm
    g = _gen(9)
    x, res = (_values(g, 4, 37, F32).requires_grad_() for _ in range(2))
    w = torch.randn(37, generator=g, device="cuda").requires_grad_()
    a, b = _values(g, 4, 37, F32), _values(g, 4, 37, F32)
    y, h = norm.add_rms_norm(x, res, w, eps=1e-3)
    grads = torch.autograd.grad((y * a).sum() + (h * b).sum(), (x, res, w))

    def loss(x, res, w):
        h = x + res
        return ((h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-3) * w) * a.double()).sum() + (h * b.double()).sum()

    at = [t.detach().double() for t in (x, res, w)]
    for i, got in enumerate(grads):
        for j in range(0, got.numel(), 5):
            hi, lo = at[i].clone(), at[i].clone()
            hi.view(-1)[j] += 1e-4
            lo.view(-1)[j] -= 1e-4
            slope = (loss(*at[:i], hi, *at[i + 1:]) - loss(*at[:i], lo, *at[i + 1:])) / 2e-4
            assert abs(float(got.reshape(-1)[j]) - float(slope)) <= 2e-5 * (1 + abs(float(slope)) + float(got.abs().max()))


def test_what_is_not_finite_stays_in_its_row(cuda):
    from engraft_ngram_amd import norm
    g = _gen(10)
    x, res = _values(g, 6, 600, F32), _values(g, 6, 600, F32)
    x[1, 3], res[4, 599] = float("nan"), float("inf")
    clean = torch.tensor([0, 2, 3, 5], device="cuda")
    y, _, _ = norm.add_rms_norm_stats(x, res, None)
    want = norm.add_rms_norm_stats(x[clean], res[clean], None)[0]
    assert torch.equal(y[clean], want) and bool(y[1].isnan().all()) and bool(y[4, 599].isnan())
    y8, _ = norm.add_rms_norm(x, res, None, out_dtype="fp8")
    assert torch.equal(y8.dequantize(F32)[clean], norm.add_rms_norm(x[clean], res[clean], None, out_dtype="fp8")[0].dequantize(F32))


def test_normed_product(cuda):
    """The norm in blocks and the product of them as one: the parts' bits, and the parts' gradients."""
    from engraft_ngram_amd import fp8, norm
    g = _gen(11)
    for m in (3, 20, 150):
        w = fp8.quantize_weight(_values(g, 300, 520, F32, 0.05))
        x, res = _values(g, m, 520, BF16).requires_grad_(), _values(g, m, 520, BF16).requires_grad_()
        nw = torch.randn(520, generator=g, device="cuda").requires_grad_()
        y, h = norm.normed_product(x, res, nw, w)
        with torch.no_grad():
            rows, h2 = norm.add_rms_norm(x, res, nw, out_dtype="fp8")
            assert torch.equal(fp8.product(rows, w), y) and torch.equal(h, h2)
            assert torch.equal(norm.normed_product(x, res, nw, w)[0], y)
            _, _, rstd = norm.add_rms_norm_stats(x, res, nw)
        d_y, d_h = _values(g, m, 300, BF16), _values(g, m, 520, BF16)
        gx, gr, gw = torch.autograd.grad((y, h), (x, res, nw), (d_y, d_h), retain_graph=True)
        want, want_w = norm.add_rms_norm_grad(fp8.product_grad(d_y, w, dtype=F32), h.detach(), rstd, nw.detach(), d_residual=d_h)
        assert torch.equal(gx, want) and torch.equal(gr, want) and torch.equal(gw, want_w)
        assert torch.equal(torch.autograd.grad(h, x, d_h)[0], d_h)
    alone = norm.normed_product(x.detach(), None, nw.detach(), w)
    assert torch.equal(alone, fp8.product(norm.rms_norm(x.detach(), nw.detach(), out_dtype="fp8"), w))


def test_rows_of_wider_buffers(cuda):
    from engraft_ngram_amd import norm
    g = _gen(12)
    x, res = _values(g, 20, 301, BF16), _values(g, 20, 301, BF16)
    wide = torch.full((20, 900), float("nan"), dtype=BF16, device="cuda")
    wide[:, 1:302], wide[:, 500:801] = x, res
    a = norm.add_rms_norm(x, res, None)
    b = norm.add_rms_norm(wide[:, 1:302], wide[:, 500:801], None)
    c = norm.add_rms_norm(x.T.contiguous().T, res, None)
    for other in (b, c):
        assert torch.equal(a[0], other[0]) and torch.equal(a[1], other[1])
    one = norm.add_rms_norm(x[:1].expand(20, 301), res, None)
    assert torch.equal(one[1], norm.add_rms_norm(x[:1].repeat(20, 1), res, None)[1])


def test_no_rows_and_rows_past_2_gib(cuda):
    from engraft_ngram_amd import fp8, norm
    none = torch.zeros((0, 300), device="cuda")
    y, h = norm.add_rms_norm(none, none, torch.ones(300, device="cuda"))
    assert y.shape == (0, 300) and h.shape == (0, 300)
    y, h = norm.add_rms_norm(none, none, None, out_dtype="fp8")
    assert y.shape == (0, 300) and y.dequantize().shape == (0, 300)
    w = fp8.quantize_weight(torch.ones((7, 300), device="cuda"))
    assert norm.normed_product(none, none, None, w)[0].shape == (0, 7)
    g = _gen(14)
    x = torch.zeros((1_700_000, 2560), dtype=BF16, device="cuda")
    x[-50:] = _values(g, 50, 2560, BF16)
    want = norm.add_rms_norm_stats(x[-50:], x[-50:], None)
    y, h, rstd = norm.add_rms_norm_stats(x, x, None)
    assert torch.equal(y[-50:], want[0]) and torch.equal(h[-50:], want[1]) and not bool(y[:-50].any())
    d_h, _ = norm.add_rms_norm_grad(y, h, rstd, None)
    assert torch.equal(d_h[-50:], norm.add_rms_norm_grad(*want, None)[0])
    y8, _ = norm.add_rms_norm(x, x, None, out_dtype="fp8")
    assert torch.equal(y8.dequantize()[-50:], norm.add_rms_norm(x[-50:], x[-50:], None, out_dtype="fp8")[0].dequantize())


def test_graphs(cuda):
    from engraft_ngram_amd import norm
    g = _gen(13)
    x, res, d_y = _values(g, 50, 700, F32), _values(g, 50, 700, F32), _values(g, 50, 700, F32)
    w = torch.randn(700, generator=g, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h, rstd = norm.add_rms_norm_stats(x, res, w)
        d_h, d_w = norm.add_rms_norm_grad(d_y, h, rstd, w)
    for _ in range(3):
        x.copy_(_values(g, 50, 700, F32))
        d_y.copy_(_values(g, 50, 700, F32))
        graph.replay()
        torch.cuda.synchronize()
        e_y, e_h, e_rstd = norm.add_rms_norm_stats(x, res, w)
        e = norm.add_rms_norm_grad(d_y, e_h, e_rstd, w)
        assert torch.equal(y, e_y) and torch.equal(h, e_h) and torch.equal(d_h, e[0]) and torch.equal(d_w, e[1])


@pytest.mark.parametrize("value", [1.0, 3.0, 5.0, 7.0, 11.0, 0.375, -13.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [2560, 1000])
def test_blocks_round_as_the_exact_rows(cuda, value, dtype, d):
    """Rows of one value are the weight itself (times its sign), however 1 / value rounds: weights on the borders between
    two e4m3 numbers, the floats beside them, and blocks whose largest is 448 2^e or the float behind it."""
    from engraft_ngram_amd import fp8, norm
    g = torch.Generator().manual_seed(3)
    w = (torch.randint(16, 32, (d,), generator=g) / 16) * 2.0 ** torch.randint(-3, 3, (d,), generator=g)
    w[::128] = 1.75 * 2.0 ** torch.randint(3, 5, (w[::128].numel(),), generator=g)
    bits = w.view(torch.int32) + torch.randint(-1, 2, (d,), generator=g, dtype=torch.int32)
    w = (bits.view(torch.float32) * (1 - 2 * torch.randint(0, 2, (d,), generator=g))).to(cuda)
    y = norm.rms_norm(torch.full((5, d), value, dtype=dtype, device=cuda), w, eps=0.0, out_dtype="fp8")
    want = fp8.quantize_rows((w if value > 0 else -w).expand(5, d).contiguous())
    assert torch.equal(y.q.view(torch.uint8), want.q.view(torch.uint8))
    assert torch.equal(y.scales.view(torch.uint8), want.scales.view(torch.uint8))
