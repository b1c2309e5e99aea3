"""Gradients that are parts of one buffer, and one that is given twice, on the GPU."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_clip import _gen, check

pytestmark = pytest.mark.gpu


def test_parts_of_one_buffer(cuda):
    """Neighbouring columns and rows, in place and into neighbouring outputs."""
    from engraft_ngram_amd import clip
    whole = torch.randn((60, 200), generator=_gen(1), device="cuda")
    kept = whole.clone()
    parts = [whole[:20, :50], whole[:20, 50:], whole[20:21], whole[21:, 100:], whole[21:, :100]]
    out = torch.empty_like(whole)
    outs = [out[:20, :50], out[:20, 50:], out[20:21], out[21:, 100:], out[21:, :100]]
    n = clip.clip_grads(parts, 3.0, out=outs)
    assert torch.equal(whole, kept)
    check([out], [kept], n, 3.0)
    assert torch.equal(clip.clip_grads(parts, 3.0), n) and torch.equal(whole, out)


def test_a_gradient_given_twice(cuda):
    """Refused where gradients are clipped; in a norm alone it counts as often as it is given."""
    from engraft_ngram_amd import clip
    x, y = torch.randn(1000, device="cuda"), torch.randn(30, device="cuda")
    kept = x.clone()
    out = [torch.empty_like(t) for t in (x, y, x)]
    for call in (lambda: clip.clip_grads([x, y, x], 1.0, out=out), lambda: clip.clip_grads([x, y, x], 1.0),
                 lambda: clip.clip_grads([x, y, x[10:20]], 1.0, out=[*out[:2], torch.empty(10, device="cuda")])):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    assert torch.equal(x, kept)
    want = math.sqrt(2 * float(x.double().square().sum()) + float(y.double().square().sum()))
    assert abs(float(clip.grad_norm([x, y, x])) - want) <= want * 2.0 ** -23
