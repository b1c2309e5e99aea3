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
