"""Values of the losses (``losses``) where they are hard to get: terms of no weight beside infinities, margins and
KL terms without end, losses that nearly cancel, gradients that overlap what they are made from.  The formulas are in
64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_losses import ALL, assert_within, lp_error, make, memory_returned, plain  # noqa: F401

pytestmark = pytest.mark.gpu


def test_overlapping_gradients_are_refused(cuda):
    """The gradient may lie in the logits' place or apart from them, also between their rows, but over none of them
    elsewhere, and over no other argument."""
    from engraft_ngram_amd import losses
    v, n = 100, 6
    buf = torch.randn(n + 1, 2 * v, device=cuda)
    t, a = torch.zeros(n, dtype=torch.int64, device=cuda), torch.zeros(n, device=cuda)
    z = buf[:n, :v]
    seg, ref = torch.arange(n, device=cuda), torch.zeros(n, device=cuda)
    wide = torch.zeros((n, v + n), device=cuda)
    kept = buf.clone()
    for out in (buf[1:, :v], buf[:n, 1:v + 1], buf[:n, v - 1:2 * v - 1], buf.view(-1)[:n * v].view(n, v),
                buf.view(-1)[v - 1:v - 1 + n * v].view(n, v)):
        for call in (lambda: losses.policy_loss_grad(z, t, a, out=out), lambda: losses.preference_loss_grad(z, t, seg, ref, out=out)):
            with pytest.raises(ValueError, match="overlap|row stride"):
                call()
    for call in (lambda: losses.policy_loss_grad(z, t, wide.view(-1)[:n], out=wide[:, :v]),
                 lambda: losses.policy_loss_grad(z, t, a, wide[0, 3:3 + n], out=wide[:, :v]),
                 lambda: losses.preference_loss_grad(z, t, seg, wide[0, 3:3 + n], out=wide[:, :v])):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert torch.equal(buf, kept)
    for call in (lambda **k: losses.policy_loss_grad(z, t, a + 1.0, **k), lambda **k: losses.preference_loss_grad(z, t, seg, ref, **k)):
        want = call()[1]
        assert torch.equal(call(out=buf[:n, v:])[1], want)
        assert torch.equal(call(out=buf[:n, v:v + v])[1], want) and torch.equal(z, kept[:n, :v])
