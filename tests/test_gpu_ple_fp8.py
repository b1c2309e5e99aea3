"""The PLE block with its projections on 8-bit blocks (``ple_forward(gemm="fp8")``): the fp32 oracle's block of the rounded
embeddings and weights, and the gradients of rounded factors, on the GPU."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle import ple as P
from tests import fp8_util as O
from tests.test_oracle_ple import ple_weights

pytestmark = pytest.mark.gpu


def _hp(hc, n):
    class HP:
        hc_mult, n_embd, f_norm_rms_eps, ple_ngram_size = hc, n, 1e-6, 3
    return HP


def _setup(hc, n, t, cuda, seed=3):
    from engraft_ngram_amd.ple import PleWeights
    w = ple_weights(hc, n, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    emb, hidden = torch.randn((t, n), generator=g) * 0.1, torch.randn((t, hc, n), generator=g) * 0.1
    return w, PleWeights(**{k: v.to(cuda) for k, v in w.items()}), emb, hidden


def _rounded(w):
    """The weights whose projections are what their blocks stand for."""
    both = O.rows(torch.cat([w["w_key"], w["w_value"]]), 128)[0].float()
    rows = w["w_key"].shape[0]
    if rows % 128:
        return dict(w, w_key=O.rows(w["w_key"], 128)[0].float(), w_value=O.rows(w["w_value"], 128)[0].float())
    return dict(w, w_key=both[:rows], w_value=both[rows:])


@pytest.mark.parametrize("hc,n,t", [(4, 2560, 1), (4, 2560, 20), (4, 2560, 90), (2, 192, 40), (1, 100, 5)])
def test_forward_is_the_rounded_block(cuda, hc, n, t):
    """Products of rounded operands are exact and their sums fp32, so the block is within the fp32 path's bars of the oracle."""
    from engraft_ngram_amd import ple
    w, wd, emb, hidden = _setup(hc, n, t, cuda)
    want, hist, s, gate = P.ple_forward(O.rows(emb)[0].float(), hidden, _rounded(w), torch.zeros(0, hc, n), hc, n, 1e-6, 3)
    diag = {}
    got, got_hist = ple.ple_forward(emb.to(cuda), hidden.to(cuda), wd, torch.zeros(0, hc, n, device=cuda), _hp(hc, n), diag=diag,
                                    gemm="fp8")
    assert float((got.cpu() - want).abs().max()) <= 1e-4
    assert float((got_hist.cpu() - hist).abs().max()) <= 1e-5
    assert float((diag["gate"].cpu() - gate).abs().max()) <= 1e-5 and float((diag["s"].cpu() - s).abs().max()) <= 1e-4


def _block(key, value, hidden, w, hc, n):
    """The block behind its projections, from an empty history, in the tensors' own type."""
    def rms(x, g):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * g.reshape(hc, n)

    t = hidden.shape[0]
    s = (rms(key.reshape(t, hc, n), w["norm_key"]) * rms(hidden, w["norm_query"])).sum(-1) / n ** 0.5
    gate = torch.sigmoid(torch.sign(s) * torch.sqrt(s.abs().clamp_min(1e-6)))
    gated = value[:, None] * gate[..., None]
    x = rms(gated, w["norm_conv"]).reshape(t, hc * n)
    acc = sum(F.pad(x, (0, 0, 3 * back, 0))[:t] * w["conv1d"][:, 3 - back] for back in range(4))
    return hidden + gated + F.silu(acc).reshape(t, hc, n)


@pytest.mark.parametrize("hc,n,t", [(4, 2560, 5), (4, 2560, 80), (2, 192, 40)])
@pytest.mark.parametrize("weights", [False, True])
def test_gradients_of_rounded_factors(cuda, hc, n, t, weights):
    """d_emb is the rounded d_key and d_value times the rounded weights; the weights' own gradients are of unrounded factors.
    d_key and d_value come from a float64 block at the kernels' key and value; theirs differ from them by up to 1e-4 of
    their largest entry, and a value that near a border between two e4m3 numbers may round the other way, by 2^-3 of itself:
    about 1e-4 / 2^-3 of the values do, which is 3e-2 2^-3 of the result's 2-norm."""
    from engraft_ngram_amd import ple
    w, wd, emb, hidden = _setup(hc, n, t, cuda, seed=9)
    r = torch.randn((t, hc, n), generator=torch.Generator().manual_seed(1)).to(cuda)
    if weights:
        for x in vars(wd).values():
            x.requires_grad_()
    e, h = emb.to(cuda).requires_grad_(), hidden.to(cuda).requires_grad_()
    out, _ = ple.ple_forward(e, h, wd, torch.zeros(0, hc, n, device=cuda), _hp(hc, n), gemm="fp8")
    (out * r).sum().backward()

    w64 = {k: v.to(cuda).double() for k, v in _rounded(w).items()}
    ev = O.rows(emb.to(cuda))[0]
    key, value = (ev @ w64["w_key"].T).requires_grad_(), (ev @ w64["w_value"].T).requires_grad_()
    h64 = hidden.to(cuda).double().requires_grad_()
    leaves = {k: w64[k].requires_grad_() for k in ("norm_key", "norm_query", "norm_conv", "conv1d")}
    (_block(key, value, h64, {**w64, **leaves}, hc, n) * r.double()).sum().backward()
    kv = O.rows(torch.cat([key.grad, value.grad], 1))[0]
    if (hc * n) % 128:
        kv = torch.cat([O.rows(key.grad)[0], O.rows(value.grad)[0]], 1)
    want = kv @ torch.cat([w64["w_key"], w64["w_value"]]).detach()
    assert float((e.grad.double() - want).norm() / want.norm()) <= 4e-3
    assert float((h.grad.double() - h64.grad).abs().max()) <= 1e-4 * float(h64.grad.abs().max())
    if weights:
        for got, exact in ((wd.w_key.grad, key.grad.T @ emb.to(cuda).double()), (wd.w_value.grad, value.grad.T @ emb.to(cuda).double()),
                           *((getattr(wd, k).grad, x.grad) for k, x in leaves.items())):
            assert float((got.double() - exact).abs().max()) <= 2e-4 * float(exact.abs().max())


@pytest.mark.parametrize("hc,n,t", [(4, 256, 40), (2, 192, 9), (1, 100, 5)])
@pytest.mark.parametrize("detach", [{}, {"detach_gate": True}, {"detach_value": True}])
def test_kept_blocks(cuda, hc, n, t, detach):
    """The same values and gradients as from the weights' own blocks, which are taken in the call; without the weights."""
    from engraft_ngram_amd import ple
    _, wd, emb, hidden = _setup(hc, n, t, cuda)
    hist = torch.zeros(0, hc, n, device=cuda)
    blocks = ple.quantize_projections(wd)
    results = []
    for w, kept in ((wd, None), (wd, blocks), (ple.PleWeights(**dict(vars(wd), w_key=None, w_value=None)), blocks)):
        e, h = emb.to(cuda).requires_grad_(), hidden.to(cuda).requires_grad_()
        out, new = ple.ple_forward(e, h, w, hist, _hp(hc, n), gemm="fp8", blocks=kept, **detach)
        out.square().sum().backward()
        with torch.no_grad():
            assert torch.equal(out, ple.ple_forward(e, h, w, hist, _hp(hc, n), gemm="fp8", blocks=kept, **detach)[0])
        results.append((out.detach(), new, e.grad, h.grad))
    for got in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, results[0]))


def test_no_positions(cuda):
    from engraft_ngram_amd import ple
    _, wd, _, _ = _setup(2, 128, 1, cuda)
    for blocks in (None, ple.quantize_projections(wd)):
        e = torch.zeros(0, 128, device=cuda, requires_grad=True)
        h = torch.zeros(0, 2, 128, device=cuda, requires_grad=True)
        hist = torch.randn(9, 2, 128, device=cuda, requires_grad=True)
        out, new = ple.ple_forward(e, h, wd, hist, _hp(2, 128), gemm="fp8", blocks=blocks)
        assert out.shape == (0, 2, 128) and torch.equal(new, hist)
        (out.sum() + new.sum()).backward()
        assert e.grad.shape == (0, 128) and torch.equal(hist.grad, torch.ones_like(hist))


def test_kept_blocks_captured(cuda):
    """A step with kept blocks, forward and gradient, replayed on other inputs beside eager work."""
    from engraft_ngram_amd import ple
    _, wd, emb, hidden = _setup(4, 256, 70, cuda)
    blocks = ple.quantize_projections(wd)
    w = ple.PleWeights(**dict(vars(wd), w_key=None, w_value=None))
    hist = torch.zeros(0, 4, 256, device=cuda)
    e, h = emb.to(cuda), hidden.to(cuda)

    def step():
        x = e.detach().requires_grad_()
        out, _ = ple.ple_forward(x, h, w, hist, _hp(4, 256), gemm="fp8", blocks=blocks)
        return out.detach(), torch.autograd.grad(out, x, torch.ones_like(out))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        e.add_(0.01 * (i + 1))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_weights_modified_in_place_are_taken_again(cuda):
    """Without kept blocks each call takes the weights' own, a captured one at each replay."""
    from engraft_ngram_amd import ple
    w, wd, emb, hidden = _setup(4, 256, 10, cuda)
    e, h, hist = emb.to(cuda), hidden.to(cuda), torch.zeros(0, 4, 256, device=cuda)
    first = ple.ple_forward(e, h, wd, hist, _hp(4, 256), gemm="fp8")[0]
    assert torch.equal(first, ple.ple_forward(e, h, wd, hist, _hp(4, 256), gemm="fp8")[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ple.ple_forward(e, h, wd, hist, _hp(4, 256), gemm="fp8")[0]
    for _ in range(3):
        wd.w_key.mul_(0.5)
        wd.w_value.add_(0.01)
        want = ple.ple_forward(e, h, wd, hist, _hp(4, 256), gemm="fp8")[0]
        graph.replay()
        torch.cuda.synchronize()
        assert not torch.equal(want, first) and torch.equal(captured, want)


def test_what_is_refused(cuda):
    from engraft_ngram_amd import ple
    w, wd, emb, hidden = _setup(5, 64, 4, cuda)
    hist = torch.zeros(0, 5, 64, device=cuda)
    ple.ple_forward(emb.to(cuda), hidden.to(cuda), wd, hist, _hp(5, 64), gemm="fp8")
    with pytest.raises(ValueError, match="fp8"):
        ple.ple_forward(emb.to(cuda).requires_grad_(), hidden.to(cuda), wd, hist, _hp(5, 64), gemm="fp8")
    with pytest.raises(ValueError, match="fp8"):
        ple.ple_forward(emb.to(cuda), hidden.to(cuda), wd, hist, _hp(5, 64), gemm="int8")
    e, h = emb.to(cuda).requires_grad_(), hidden.to(cuda)
    with torch.no_grad():  # parameters, without a gradient
        ple.ple_forward(e, h, wd, hist, _hp(5, 64), gemm="fp8")
    blocks = ple.quantize_projections(wd, transpose=False)
    ple.ple_forward(e.detach(), h, wd, hist, _hp(5, 64), gemm="fp8", blocks=blocks)
    with pytest.raises(ValueError, match="blocks"):
        ple.ple_forward(e.detach(), h, wd, hist, _hp(5, 64), blocks=blocks)
    none = ple.PleWeights(**dict(vars(wd), w_key=None))
    with pytest.raises(ValueError, match="blocks"):
        ple.ple_forward(e.detach(), h, none, hist, _hp(5, 64), gemm="fp8")
    _, w2, emb2, hidden2 = _setup(2, 64, 4, cuda)
    with pytest.raises(ValueError, match="blocks"):
        ple.ple_forward(emb2.to(cuda), hidden2.to(cuda), w2, torch.zeros(0, 2, 64, device=cuda), _hp(2, 64), gemm="fp8", blocks=blocks)
    half = ple.quantize_projections(w2, transpose=False)
    with pytest.raises(ValueError, match="transpose"):
        ple.ple_forward(emb2.to(cuda).requires_grad_(), hidden2.to(cuda), w2, torch.zeros(0, 2, 64, device=cuda), _hp(2, 64),
                        gemm="fp8", blocks=half)
