"""Orthogonalised updates (``muon``) of weights: every value of the weights after a step, the large
products' kernels, steps that fail, outputs that overlap, norms at the type's ends.  The formulas are
``test_gpu_muon.plain``'s, in 64 bits; X's tolerance is derived there."""
from __future__ import annotations

import math
import re

import pytest
import torch

from tests.conftest import ROOT
from tests.test_gpu_muon import ROUNDING, memory_returned, off, plain, random  # noqa: F401

pytestmark = pytest.mark.gpu


def half_unit(x, dtype):
    """Half a unit in the last place of `dtype` at float64 x (normal numbers)."""
    bits = {torch.float32: 24, torch.bfloat16: 8, torch.float16: 11}[dtype]
    return torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent - 1 - bits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(64, 256), (130, 70), (200, 300), (700, 520)])
def test_every_weight(cuda, shape, dtype):
    """Weights of every type take the update of fp32 accuracy: each is the 64-bit result rounded once, but for
    lr scale 64 2^-23 where that moves it over a rounding's edge (|X_ij| <= 1.2, and a value's share of
    X's error is far below the whole)."""
    from engraft_ngram_amd import muon
    lr, decay = 0.2, 0.1
    w, g = random(shape, dtype, 1, 0.02), random(shape, dtype, 2)
    new = w.clone()
    muon.muon_step([new], [g], [torch.zeros(shape, device=cuda)], lr=lr, weight_decay=decay)
    rate = lr * math.sqrt(max(1.0, shape[0] / shape[1]))
    want = (1 - lr * decay) * w.double() - rate * plain(1.95 * g.double())
    tol = half_unit(want, dtype) + rate * 64 * 2.0 ** -23 + 2.0 ** -24 * want.abs()
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # below the smallest normal number
    assert ((new.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("wt", [torch.float16, torch.float32])
def test_two_planes_step(cuda, wt):
    """Three products in a step of f16 weights as of f32 ones: two steps, to 64 2^-23 of X besides the weights' rounding."""
    from engraft_ngram_amd import muon
    lr, shape = 0.05, (96, 200)
    w, m = random(shape, wt, 1, 0.1), torch.zeros(shape, device=cuda)
    want_w, want_m, tol = w.double(), m.double(), 0.0
    for step in range(2):
        g = random(shape, torch.float32, 20 + step, 1e-3)
        muon.muon_step([w], [g], [m], lr=lr, momentum=0.9)
        want_m = 0.9 * want_m + g.double()
        x = plain(g.double() + 0.9 * want_m)
        want_w = want_w - lr * x
        tol = tol + lr * 64 * 2.0 ** -23 * x.norm() + 2 * ROUNDING[wt] * want_w.norm()
        assert (w.double() - want_w).norm() <= tol


# ---- the products of 128 x 128 tiles ------------------------------------------------------------

def tiles(shape, count=1):
    """128 x 128 tiles of (a symmetric product, the step's product)."""
    m, n = sorted(-(-x // 64) * 64 for x in shape)
    m, n = -(-m // 128), -(-n // 128)
    return count * m * (m + 1) // 2, count * m * n


def limits():
    """(few, many): the tile counts between which products take 128 x 128 tiles of four wavefronts."""
    text = (ROOT / "engraft-ngram_amd" / "csrc" / "eg_muon.hip").read_text()
    found = re.search(r"kFewTiles = (\d+), kManyTiles = (\d+);", text)
    return int(found[1]), int(found[2])


@pytest.mark.parametrize("products", ["fp16x3", "fp16"])
@pytest.mark.parametrize("shape", [(2113, 2177), (2177, 2113), (2000, 3000), (3000, 2000)])
def test_large_tiles(cuda, shape, products):
    """Products of more than kFewTiles tiles, partial last tiles among them, wide and tall: X, and a step of
    weights inside a padded buffer, nothing of which is written outside."""
    from engraft_ngram_amd import muon
    few, many = limits()
    assert few < tiles(shape)[0] and tiles(shape)[1] < many
    u = 2.0 ** -23 if products == "fp16x3" else 2.0 ** -12
    for dtype in (torch.float32, torch.bfloat16):
        x = random(shape, dtype, 7)
        want = plain(x)
        got = muon.orthogonalize(x, products=products)
        assert off(got, want) <= 64 * u + ROUNDING[dtype], (dtype, off(got, want))
        assert torch.equal(got, muon.orthogonalize(x, products=products))
        buf = torch.full((shape[0] + 2, shape[1] + 7), 7.0, dtype=dtype, device=cuda)
        w = buf[1:-1, 3:-4]
        w.copy_(random(shape, dtype, 8, 0.02))
        before = w.double()
        muon.muon_step([w], [x], [torch.zeros(shape, device=cuda)], lr=0.1, momentum=0.0, products=products)
        rate = 0.1 * math.sqrt(max(1.0, shape[0] / shape[1]))
        new = before - rate * want
        assert (w.double() - new).norm() <= rate * 64 * u * want.norm() + ROUNDING[dtype] * new.norm()
        w.fill_(7.0)
        assert (buf == 7.0).all()


@pytest.mark.parametrize("products", ["fp16x3", "fp16"])
@pytest.mark.parametrize("shape", [(800, 1030), (1030, 800)])
def test_many_tiles(cuda, shape, products):
    """A batch whose step's product has at least kManyTiles tiles (one wavefront a tile with one plane): the first,
    a middle and the last matrix against the formula, every one against its own call in smaller tiles."""
    from engraft_ngram_amd import muon
    few, many = limits()
    count = 24
    assert few < tiles(shape, count)[0] and many <= tiles(shape, count)[1] and tiles(shape)[1] <= few
    u = 2.0 ** -23 if products == "fp16x3" else 2.0 ** -12
    x = random((count, *shape), torch.bfloat16, 9)
    got = torch.full(x.shape, 7.0, device=cuda)
    muon.orthogonalize(x, out=got, products=products)
    for i in range(count):
        if i in (0, 11, count - 1):
            assert off(got[i], plain(x[i])) <= 64 * u, off(got[i], plain(x[i]))
        one = torch.empty(shape, device=cuda)
        muon.orthogonalize(x[i], out=one, products=products)
        assert off(got[i], one.double()) <= 128 * u


def test_norm_of_many_parts(cuda):
    """A matrix of some thousand 64 x 64 tiles: its norm is the sum of as many parts, taken by the workgroups that use it
    or, above kOwnSumTiles, in a launch of its own."""
    from engraft_ngram_amd import muon
    own = int(re.search(r"kOwnSumTiles = (\d+);", (ROOT / "engraft-ngram_amd" / "csrc" / "eg_muon.hip").read_text())[1])
    assert 66_000 // 64 < own < 300_001 // 64
    for shape in ((40, 300_001), (300_001, 40), (64, 66_000)):
        x = random(shape, torch.float32, 10)
        assert off(muon.orthogonalize(x, steps=1), plain(x, steps=1)) <= 64 * 2.0 ** -23


@pytest.mark.parametrize("shape", [(70, 90), (200, 300)])
@pytest.mark.parametrize("size", [1e-32, 1e-25, 1e-21, 1e21, 1e30, 1e37])
def test_norms_whose_squares_leave_fp32(cuda, shape, size):
    """|u|^2 below fp32's smallest number or above its largest: the same direction."""
    from engraft_ngram_amd import muon
    x = random(shape, torch.float32, 11, size)
    got = muon.orthogonalize(x, eps=1e-34)
    assert off(got, plain(x, eps=1e-34)) <= 64 * 2.0 ** -23
    zeros = torch.zeros(shape, device=cuda)
    assert (muon.orthogonalize(zeros, eps=1e-34) == 0).all()


# ---- steps that are refused ---------------------------------------------------------------------

def test_a_step_is_whole_or_not_at_all(cuda):
    """Matrices of a shape that is refused beside others: no weight, momentum or version of any is touched;
    and a step counts as a version of each weight and momentum."""
    from engraft_ngram_amd import muon
    w, m = random((8, 8), torch.float32, 1), random((8, 8), torch.float32, 2)
    far = torch.zeros(((1 << 20) + 1, 1), device=cuda)
    before = w.clone(), m.clone(), w._version, m._version, far._version
    state = muon.MuonState([w, far], [m, torch.zeros_like(far)])
    for weights in ([0, 1], [1, 0]):
        params, momenta = [(w, far)[i] for i in weights], [(m, state.momenta[1])[i] for i in weights]
        with pytest.raises(ValueError, match="2\\^20"):
            muon.muon_step(params, [torch.ones_like(p) for p in params], momenta, lr=0.1)
    with pytest.raises(ValueError, match="2\\^20"):
        state.step([torch.ones_like(w), torch.ones_like(far)], lr=0.1)
    assert torch.equal(w, before[0]) and torch.equal(m, before[1]) and state.step_count == 0
    assert (w._version, m._version, far._version) == before[2:]
    # a rate that overflows for the tall shape alone
    tall = torch.zeros((4000, 1), device=cuda)
    with pytest.raises(ValueError, match="not finite"):
        muon.muon_step([w, tall], [w.clone(), tall.clone()], [m, tall.clone()], lr=1e37)
    assert torch.equal(w, before[0]) and torch.equal(m, before[1])
    muon.muon_step([w, tall], [w.clone(), tall.clone()], [m, torch.zeros_like(tall)], lr=0.1)
    assert w._version > before[2] and m._version > before[3]


def test_memory_for_the_step_is_had_before_it(cuda):
    """A workspace that torch's allocator refuses for the last shape leaves the first one's weights alone."""
    from engraft_ngram_amd import muon
    w, m = random((8, 8), torch.float32, 1), random((8, 8), torch.float32, 2)
    big = torch.zeros((4096, 4096), device=cuda)
    before = w.clone(), m.clone(), w._version
    grads, momenta = [w.clone(), big.clone()], [m, big.clone()]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    held = torch.cuda.memory_reserved(0)
    torch.cuda.set_per_process_memory_fraction((held + (64 << 20)) / total)
    try:
        with pytest.raises(RuntimeError, match="out of memory"):
            muon.muon_step([w, big], grads, momenta, lr=0.1)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(w, before[0]) and torch.equal(m, before[1]) and w._version == before[2]


def test_workspace_is_bounded(cuda):
    """Large matrices share a launch only as far as their workspace stays within a bound; each as on its own."""
    from engraft_ngram_amd import _lib, muon
    lib = _lib.load()
    one = lib.eg_muon_workspace_size(4096, 4096, 1, 2)
    assert lib.eg_muon_workspace_size(4096, 4096, 64, 2) <= max(one, 2 << 30) < 64 * one
    x = random((3, 8192, 8192), torch.bfloat16, 12)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = muon.orthogonalize(x, steps=1, products="fp16x3")
    assert torch.cuda.max_memory_allocated() - before <= got.numel() * 2 + (2 << 30)
    for i in range(3):
        assert torch.equal(got[i], muon.orthogonalize(x[i], steps=1, products="fp16x3"))


def test_overlapping_outputs_are_refused(cuda):
    """A weight given twice, matrices that share elements, a momentum over a gradient or a weight; what only
    lies side by side, and x's own place, are taken."""
    from engraft_ngram_amd import muon
    w, g = random((60, 80), torch.float32, 1), random((60, 80), torch.float32, 2)

    def zeros(n=1):
        return [torch.zeros((60, 80), device=cuda) for _ in range(n)]

    flat = torch.zeros(20_000, device=cuda)
    rows = flat.as_strided((60, 80), (1, 1))
    m = zeros()[0]
    square = random((2, 64, 64), torch.float32, 3)
    for params, grads, momenta in (
            ([w, w], [g, g], zeros(2)), ([w, w[:, :40]], [g, g[:, :40]], [m, torch.zeros((60, 40), device=cuda)]),
            ([w, w.T], [g, g.T], [m, torch.zeros((80, 60), device=cuda)]), ([rows], [g], [m]), ([w], [g], [w]),
            ([w], [m], [m]), ([w, w + 1.0], [g, g], [m, m]), ([w], [g], [rows]),
            ([flat[:4800].view(60, 80), flat[4799:9599].view(60, 80)], [g, g], zeros(2)),
            ([w, w + 1.0], [g, w], zeros(2))):
        kept = [t.clone() for t in (*params, *momenta)]
        with pytest.raises(ValueError, match="overlap"):
            muon.muon_step(params, grads, momenta, lr=0.1)
        assert all(torch.equal(a, b) for a, b in zip(kept, (*params, *momenta)))
    over = square.view(-1)[64:64 + 4096].view(64, 64)  # of x alone: x is read whole before anything is written
    want = muon.orthogonalize(square[0])
    assert torch.equal(muon.orthogonalize(square[0], out=over), want)
    # columns of one buffer, halves of a batch, x's own place and its transpose's
    both = torch.cat([w, w + 1.0], 1)
    apart = [w.clone(), w + 1.0]
    muon.muon_step([both[:, :80], both[:, 80:]], [g, g], zeros(2), lr=0.1)
    muon.muon_step(apart, [g, g], zeros(2), lr=0.1)
    assert torch.equal(both, torch.cat(apart, 1))
    want = muon.orthogonalize(square)
    turned = square.clone()
    muon.orthogonalize(square, out=square)
    assert torch.equal(square, want)
    want = muon.orthogonalize(turned[0])
    muon.orthogonalize(turned[0], out=turned[0].T)
    assert torch.equal(turned[0].T, want)
