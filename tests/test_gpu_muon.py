"""Orthogonalised updates (``muon``) against a plain float64 implementation: shapes
from 1 x 1, odd ones, tall and wide, batches, types and strides.

Tolerance of X in the Frobenius norm.  An iteration rounds X, A and B once each
(unit u = 2^-12 for one fp16 plane, 2^-23 for two) besides fp32 sums of random sign,
about 16 roundings in five steps; rounding noise is amplified like the
singular values it meets, so relative to X it keeps its size but along the smallest
singular values of a square random matrix, a few times it.  64 u |X| covers both
(and is far below the 2^-12 |X| a missing cross product would leave in two planes'
result)."""
from __future__ import annotations

import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_returned():
    """What torch's allocator keeps of these tests' tensors goes back: other tests read its statistics."""
    yield
    import gc

    import torch
    gc.collect()
    torch.cuda.empty_cache()

ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a unit in the last place
QUINTIC = (3.4445, -4.7750, 2.0315)
SHAPES = [(1, 1), (1, 40), (40, 1), (2, 3), (31, 33), (64, 64), (65, 130), (130, 65), (128, 640), (257, 200),
          (200, 1031), (1031, 200), (384, 384), (520, 1290)]


def plain(x, steps=5, coefficients=None, eps=1e-7):
    x = x.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for a, b, c in coefficients or [QUINTIC] * steps:
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.T if tall else x


def random(shape, dtype, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("products", ["fp16x3", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(cuda, shape, products):
    from engraft_ngram_amd import muon
    for dtype, size in ((torch.float32, 1.0), (torch.bfloat16, 1e-4), (torch.float16, 30.0)):
        x = random(shape, dtype, shape[0] + shape[1], size)
        before = x.clone()
        got = muon.orthogonalize(x, products=products)
        assert got.dtype == dtype and got.shape == x.shape and torch.equal(x, before)
        want = plain(x)
        u = 2.0 ** -23 if products == "fp16x3" else 2.0 ** -12
        assert off(got, want) <= 64 * u + ROUNDING[dtype], (dtype, off(got, want))
        assert torch.equal(got, muon.orthogonalize(x, products=products))


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("wt,gt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
def test_step(cuda, wt, gt, nesterov):
    """Two steps of weights of several shapes at once: w and m against the formula.  w's error: its own
    rounding, and lr scale times X's (above); m's: three fp32 roundings a step."""
    from engraft_ngram_amd import muon
    lr, decay, mu = 0.05, 0.1, 0.9
    shapes = [(96, 200), (200, 96), (96, 200), (3, 70, 50)]
    params = [random(s, wt, i, 0.1) for i, s in enumerate(shapes)]
    momenta = [random(s, torch.float32, 10 + i, 1e-3) for i, s in enumerate(shapes)]
    state = muon.MuonState([p.clone() for p in params], [m.clone() for m in momenta], momentum=mu, nesterov=nesterov)
    want_p = [p.double() for p in params]
    want_m = [m.double() for m in momenta]
    u = 2.0 ** -23 if wt == torch.float32 else 2.0 ** -12
    tol_p = [torch.zeros((), dtype=torch.float64, device=cuda) for _ in shapes]
    for step in range(2):
        grads = [random(s, gt, 100 * step + 20 + i, 1e-3) for i, s in enumerate(shapes)]
        state.step(grads, lr=lr, weight_decay=decay)
        for i, g in enumerate(grads):
            want_m[i] = mu * want_m[i] + g.double()
            upd = g.double() + mu * want_m[i] if nesterov else want_m[i]
            rate = lr * math.sqrt(max(1.0, shapes[i][-2] / shapes[i][-1]))
            x = torch.stack([plain(q) for q in upd]) if upd.dim() == 3 else plain(upd)
            want_p[i] = (1 - lr * decay) * want_p[i] - rate * x
            tol_p[i] = tol_p[i] + rate * 64 * u * x.norm() + 2 * ROUNDING[wt] * want_p[i].norm()
            assert off(state.momenta[i], want_m[i]) <= 4 * (step + 1) * 2.0 ** -24
            assert (state.params[i].double() - want_p[i]).norm() <= tol_p[i]
            assert state.params[i].dtype == wt
    assert state.step_count == 2


def test_strides(cuda):
    """Padded rows, columns contiguous, slices of a batch: the bits of the contiguous call, and nothing
    written outside."""
    from engraft_ngram_amd import muon
    w, g, m = random((90, 150), torch.float32, 1, 0.1), random((90, 150), torch.float32, 2), random((90, 150), torch.float32, 3)
    base = [t.clone() for t in (w, m)]
    muon.muon_step([base[0]], [g], [base[1]], lr=0.1, weight_decay=0.1)

    def padded(t):
        buf = torch.full((92, 157), 7.0, device=cuda)
        buf[1:91, 3:153] = t
        return buf, buf[1:91, 3:153]

    bufs = [padded(t) for t in (w, g, m)]
    muon.muon_step([bufs[0][1]], [bufs[1][1]], [bufs[2][1]], lr=0.1, weight_decay=0.1)
    assert torch.equal(bufs[0][1], base[0]) and torch.equal(bufs[2][1], base[1])
    for buf, view in bufs:
        view.fill_(7.0)
        assert (buf == 7.0).all()
    turned = [t.T.contiguous().T for t in (w, g, m)]
    muon.muon_step([turned[0]], [turned[1]], [turned[2]], lr=0.1, weight_decay=0.1)
    assert torch.equal(turned[0], base[0]) and torch.equal(turned[2], base[1])
    every = torch.zeros((5, 90, 150), device=cuda)
    every[::2] = w
    mom = torch.stack([m, m, m])
    muon.muon_step([every[::2]], [g.expand(3, 90, 150)], [mom], lr=0.1, weight_decay=0.1)
    assert all(torch.equal(every[i], base[0]) for i in (0, 2, 4)) and (every[1::2] == 0).all()


def test_many_matrices(cuda):
    """More matrices than a launch holds: each as on its own."""
    from engraft_ngram_amd import muon
    x = random((131, 20, 36), torch.bfloat16, 5)
    got = muon.orthogonalize(x)
    for i in (0, 63, 64, 130):
        assert torch.equal(got[i], muon.orthogonalize(x[i]))


def test_extremes(cuda):
    """Zeros stay zeros (a zero update leaves the decayed weight), one element becomes the polynomial's
    value, tiny and large updates keep their direction, a NaN reaches its own matrix only."""
    from engraft_ngram_amd import muon
    x = torch.zeros((4, 70, 90), device=cuda)
    x[1, 3, 5] = -2.0
    x[2] = random((70, 90), torch.float32, 1, 1e-15)
    x[3] = random((70, 90), torch.float32, 2, 1e12)
    got = muon.orthogonalize(x, eps=1e-30)
    assert (got[0] == 0).all()
    s = 1.0
    for _ in range(5):
        s = QUINTIC[0] * s + QUINTIC[1] * s ** 3 + QUINTIC[2] * s ** 5
    assert abs(float(got[1, 3, 5]) + s) < 1e-5 and int((got[1] != 0).sum()) == 1
    for i in (2, 3):
        assert off(got[i], plain(x[i], eps=1e-30)) < 64 * 2.0 ** -23
    x[2, 0, 0] = math.nan
    got2 = muon.orthogonalize(x, eps=1e-30)
    assert got2[2].isnan().all() and torch.equal(got2[3], got[3]) and torch.equal(got2[1], got[1])
    w = random((70, 90), torch.float32, 3)
    keep = w.clone()
    muon.muon_step([w], [torch.zeros_like(w)], [torch.zeros_like(w)], lr=0.1, weight_decay=0.5)
    assert torch.allclose(w, keep * 0.95, rtol=2.0 ** -22, atol=0.0)


def test_coefficients(cuda):
    """A schedule of coefficients, one step, and the cubic iteration to an orthogonal matrix."""
    from engraft_ngram_amd import muon
    x = random((60, 100), torch.float32, 4)
    schedule = [(4.0, -6.0, 2.5), (3.0, -4.0, 1.8), (2.0, -1.5, 0.5)]
    assert off(muon.orthogonalize(x, steps=3, coefficients=schedule), plain(x, coefficients=schedule)) < 64 * 2.0 ** -23
    assert off(muon.orthogonalize(x, steps=1), plain(x, steps=1)) < 64 * 2.0 ** -23
    q = muon.orthogonalize(x, steps=25, coefficients=(1.5, -0.5, 0.0)).double()
    assert (q @ q.T - torch.eye(60, device=cuda)).norm() < 1e-4  # 25 steps of 64 * 2^-23 / 5, |I| = 8


def test_in_a_graph_and_on_another_stream(cuda):
    from engraft_ngram_amd import muon
    w0, g, m0 = random((150, 300), torch.bfloat16, 1, 0.1), random((150, 300), torch.bfloat16, 2), random((150, 300), torch.float32, 3)
    w, m = w0.clone(), m0.clone()
    wants = []
    for k in range(4):
        muon.muon_step([w], [g * (k + 1)], [m], lr=0.1)
        wants.append((w.clone(), m.clone()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    w1, m1 = w0.clone(), m0.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(2):
            muon.muon_step([w1], [g * (k + 1)], [m1], lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(w1, wants[1][0]) and torch.equal(m1, wants[1][1])
    w2, m2, g2 = w0.clone(), m0.clone(), g.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon.muon_step([w2], [g2], [m2], lr=0.1)
    w2.copy_(w0)
    m2.copy_(m0)
    for k in range(4):
        g2.copy_(g * (k + 1))
        graph.replay()
        muon.orthogonalize(random((200, 200), torch.float32, k))  # the program's own work between replays
        torch.cuda.synchronize()
        assert torch.equal(w2, wants[k][0]) and torch.equal(m2, wants[k][1])


def test_python_arguments_are_checked_on_the_gpu(cuda):
    from engraft_ngram_amd import muon
    w, m = torch.zeros((4, 6), device=cuda), torch.zeros((4, 6), device=cuda)
    for match, call in (
            ("params must be", lambda: muon.muon_step([w[0]], [w[0]], [m[0]], lr=0.1)),
            ("params must be", lambda: muon.muon_step([w.double()], [w], [m], lr=0.1)),
            ("grads must be", lambda: muon.muon_step([w], [w[:2]], [m], lr=0.1)),
            ("momenta must be f32", lambda: muon.muon_step([w], [w], [m.half()], lr=0.1)),
            ("expanded", lambda: muon.muon_step([w[:1].expand(4, 6)], [w], [m], lr=0.1)),
            ("1 params, 2 grads", lambda: muon.muon_step([w], [w, w], [m], lr=0.1)),
            ("coefficients", lambda: muon.muon_step([w], [w], [m], lr=0.1, coefficients=[(1.0, 2.0, 3.0)] * 4)),
            ("coefficients", lambda: muon.orthogonalize(w, coefficients=(1.0, 2.0))),
            ("singular values", lambda: muon.orthogonalize(w, coefficients=(90.0, 1.0, 1.0))),
            ("products", lambda: muon.orthogonalize(w, products="fp8")),
            ("eps", lambda: muon.orthogonalize(w, eps=0.0)),
            ("not finite", lambda: muon.muon_step([w], [w], [m], lr=math.inf)),
            ("out must be", lambda: muon.orthogonalize(w, out=w[:2]))):
        with pytest.raises(ValueError, match=match):
            call()
    before = w.clone()
    muon.muon_step([w[:0]], [w[:0]], [m[:0]], lr=0.1)  # nothing to do
    assert torch.equal(w, before)


def test_block_sees_the_step(cuda):
    """ple_forward keeps planes of its weights between calls: after a step of the weights (w_key as one matrix a
    stream, a view) it computes with the new ones, and autograd refuses a graph that saved the old."""
    from engraft_ngram_amd import muon, ple
    n, hc, t = 64, 4, 40
    w = ple.PleWeights(w_key=random((hc * n, n), torch.float32, 1, 0.1), w_value=random((n, n), torch.float32, 2, 0.1),
                       norm_key=torch.ones(hc * n, device=cuda), norm_query=torch.ones(hc * n, device=cuda),
                       norm_conv=torch.ones(hc * n, device=cuda), conv1d=random((hc * n, 4), torch.float32, 3, 0.1))
    w.w_key.requires_grad_()
    w.w_value.requires_grad_()
    emb, hidden = random((t, n), torch.float32, 4), random((t, hc, n), torch.float32, 5)
    hist = torch.zeros((9, hc, n), device=cuda)

    hp = types.SimpleNamespace(hc_mult=hc, n_embd=n, f_norm_rms_eps=1e-6, ple_ngram_size=3)
    before = ple.ple_forward(emb, hidden, w, hist, hp)[0]
    grads = torch.autograd.grad(before.square().sum(), [w.w_key, w.w_value], retain_graph=True)
    state = muon.MuonState([w.w_key.view(hc, n, n), w.w_value])
    state.step([grads[0].view(hc, n, n), grads[1]], lr=0.1)
    after = ple.ple_forward(emb, hidden, w, hist, hp)[0]
    fresh = ple.PleWeights(w.w_key.detach().clone(), w.w_value.detach().clone(), w.norm_key, w.norm_query, w.norm_conv,
                           w.conv1d)
    assert torch.equal(after, ple.ple_forward(emb, hidden, fresh, hist, hp)[0]) and not torch.equal(after, before)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        before.square().sum().backward()


def test_products_by_type(cuda):
    """Without `products`: f32 and f16 weights take three products, bf16 weights one; an f16 weight's update
    is then off by its own rounding alone."""
    from engraft_ngram_amd import muon
    for dtype, products in ((torch.float32, "fp16x3"), (torch.float16, "fp16x3"), (torch.bfloat16, "fp16")):
        x = random((200, 300), dtype, 6)
        assert torch.equal(muon.orthogonalize(x), muon.orthogonalize(x, products=products))
    w, g = random((90, 90), torch.float16, 7, 0.02), random((90, 90), torch.float32, 8)
    new = w.clone()
    muon.muon_step([new], [g], [torch.zeros_like(g)], lr=0.2)
    want = w.double() - 0.2 * plain(1.95 * g)
    assert ((new.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -24 + 0.2 * 64 * 2.0 ** -23).all()
