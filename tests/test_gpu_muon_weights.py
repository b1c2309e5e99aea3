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
