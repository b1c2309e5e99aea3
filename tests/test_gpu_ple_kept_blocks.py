"""Kept 8-bit blocks of the PLE block's projections that change, or whose weights do, on the GPU."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_ple_fp8 import _hp, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hc,n", [(4, 256), (1, 100)])  # key and value as one weight, and as two
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("detach", [{}, {"detach_gate": True}])
@pytest.mark.parametrize("which", ["q_t", "scales_t"])
def test_blocks_written_before_the_gradient(cuda, hc, n, weights, detach, which):
    """A gradient from other blocks than the forward's would be wrong: it is refused, as a saved tensor's is."""
    from engraft_ngram_amd import ple
    _, wd, emb, hidden = _setup(hc, n, 9, cuda)
    if weights:
        wd.norm_key.requires_grad_()
    blocks = ple.quantize_projections(wd)
    hist = torch.zeros(0, hc, n, device=cuda)

    def loss():
        e = emb.to(cuda).requires_grad_()
        return e, ple.ple_forward(e, hidden.to(cuda), wd, hist, _hp(hc, n), gemm="fp8", blocks=blocks, **detach)[0].sum()

    e, whole = loss()
    whole.backward()
    assert bool(e.grad.any())
    _, late = loss()
    getattr(blocks.parts[-1], which).view(torch.uint8).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()


def test_blocks_replaced_before_the_gradient(cuda):
    """Other tensors in the place of the forward's change nothing: its own are the gradient's."""
    from engraft_ngram_amd import ple
    _, wd, emb, hidden = _setup(4, 256, 9, cuda)
    blocks, hist, grads = ple.quantize_projections(wd), torch.zeros(0, 4, 256, device=cuda), []
    for replace in (False, True):
        e = emb.to(cuda).requires_grad_()
        out, _ = ple.ple_forward(e, hidden.to(cuda), wd, hist, _hp(4, 256), gemm="fp8", blocks=blocks)
        if replace:
            blocks.parts[0].q_t = torch.zeros_like(blocks.parts[0].q_t.view(torch.uint8)).view(torch.float8_e4m3fn)
        out.square().sum().backward()
        grads.append(e.grad)
    assert torch.equal(*grads)
