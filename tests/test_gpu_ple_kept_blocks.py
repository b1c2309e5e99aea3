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


def _weights_of(wd, **changed):
    from engraft_ngram_amd import ple
    return ple.PleWeights(**dict(vars(wd), **changed))


@pytest.mark.parametrize("hc,n", [(4, 256), (1, 100)])
def test_weights_that_are_not_the_blocks(cuda, hc, n):
    """Weights beside blocks of others would be trained, or taken to be served, without an effect: they are refused."""
    from engraft_ngram_amd import ple
    _, wd, emb, hidden = _setup(hc, n, 5, cuda)
    e, h, hist = emb.to(cuda), hidden.to(cuda), torch.zeros(0, hc, n, device=cuda)
    blocks = ple.quantize_projections(wd)

    def run(w):
        return ple.ple_forward(e, h, w, hist, _hp(hc, n), gemm="fp8", blocks=blocks)[0]

    want = run(wd)
    # the same memory at the same version, under other names, and one or none of them given
    for w in (_weights_of(wd, w_key=wd.w_key.detach().requires_grad_()), _weights_of(wd, w_value=torch.nn.Parameter(wd.w_value)),
              _weights_of(wd, w_key=None), _weights_of(wd, w_key=None, w_value=None)):
        assert torch.equal(run(w), want)
    for w in (_weights_of(wd, w_key=wd.w_key.clone()), _weights_of(wd, w_value=wd.w_value.clone().requires_grad_()),
              _weights_of(wd, w_value=wd.w_value.T)):
        with pytest.raises(ValueError, match="quantize_projections"):
            run(w)
    wd.w_value.mul_(0.5)
    with pytest.raises(ValueError, match="quantize_projections"):
        run(wd)
    assert torch.equal(run(_weights_of(wd, w_key=None, w_value=None)), want)  # they still stand for what they were made of
    blocks = ple.quantize_projections(wd)
    fresh = run(wd)
    assert not torch.equal(fresh, want)
    assert torch.equal(fresh, ple.ple_forward(e, h, wd, hist, _hp(hc, n), gemm="fp8")[0])
    # weights that are gone are no longer known
    gone = ple.quantize_projections(_weights_of(wd, w_key=wd.w_key.clone(), w_value=wd.w_value.clone()))
    with pytest.raises(ValueError, match="quantize_projections"):
        ple.ple_forward(e, h, wd, hist, _hp(hc, n), gemm="fp8", blocks=gone)


def test_blocks_follow_updated_weights(cuda):
    """A weight update by the library counts as a change; blocks taken again are the updated weights'."""
    from engraft_ngram_amd import muon, ple
    _, wd, emb, hidden = _setup(2, 256, 30, cuda)
    e, h, hist = emb.to(cuda), hidden.to(cuda), torch.zeros(0, 2, 256, device=cuda)
    blocks = ple.quantize_projections(wd)
    before = ple.ple_forward(e, h, wd, hist, _hp(2, 256), gemm="fp8", blocks=blocks)[0]
    opt = muon.MuonState([wd.w_key, wd.w_value])
    opt.step([torch.randn_like(wd.w_key), torch.randn_like(wd.w_value)], lr=1e-2)
    with pytest.raises(ValueError, match="quantize_projections"):
        ple.ple_forward(e, h, wd, hist, _hp(2, 256), gemm="fp8", blocks=blocks)
    after = ple.ple_forward(e, h, wd, hist, _hp(2, 256), gemm="fp8", blocks=ple.quantize_projections(wd))[0]
    assert not torch.equal(after, before)
    assert torch.equal(after, ple.ple_forward(e, h, wd, hist, _hp(2, 256), gemm="fp8")[0])


def test_weights_without_versions(cuda):
    """Inference tensors have no version; their blocks serve beside them."""
    from engraft_ngram_amd import ple
    with torch.inference_mode():
        _, wd, emb, hidden = _setup(2, 256, 3, cuda)
        hist = torch.zeros(0, 2, 256, device=cuda)
        args = (emb.to(cuda), hidden.to(cuda), wd, hist, _hp(2, 256))
        blocks = ple.quantize_projections(wd)
        assert torch.equal(ple.ple_forward(*args, gemm="fp8", blocks=blocks)[0], ple.ple_forward(*args, gemm="fp8")[0])
