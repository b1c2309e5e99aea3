"""The 8-bit operators together, as a training step uses them: rows through the PLE block on 8-bit projections, the residual's
norm into an 8-bit head, a policy loss of its logits, the gradients clipped as one, and the weights' updates."""
from __future__ import annotations

import pytest
import torch

from tests import fp8_util as O

pytestmark = pytest.mark.gpu

HC, N, T, VOCAB = 2, 256, 60, 700


class HP:
    hc_mult, n_embd, f_norm_rms_eps, ple_ngram_size = HC, N, 1e-6, 3


class _Product(torch.autograd.Function):
    """Rounded factors forward, and in the gradient."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(w)
        return O.rows(x)[0] @ w.T

    @staticmethod
    def backward(ctx, d):
        return O.rows(d)[0] @ ctx.saved_tensors[0], None


def test_a_step(cuda):
    from engraft_ngram_amd import clip, fp8, losses, muon, norm, ple
    g = torch.Generator(device="cuda").manual_seed(1)

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    w = ple.PleWeights(randn(HC * N, N, scale=0.06), randn(N, N, scale=0.06), randn(HC * N), randn(HC * N), randn(HC * N),
                       randn(HC * N, 4, scale=0.3))
    head = fp8.quantize_weight(randn(VOCAB, N, scale=0.06))
    norm_weight, emb, hidden = randn(N), randn(T, N), randn(T, HC, N)
    leaves = [emb, norm_weight, *vars(w).values()]
    for x in leaves:
        x.requires_grad_()
    targets = torch.randint(0, VOCAB, (T,), generator=g, device="cuda")
    advantages = randn(T)

    out, _ = ple.ple_forward(emb, hidden, w, torch.zeros(0, HC, N, device="cuda"), HP, gemm="fp8")
    mixed = (out - hidden).mean(1).detach().requires_grad_()  # the block's own output, and a stream's residual
    residual = hidden[:, 0].clone().requires_grad_()
    logits, h = norm.normed_product(mixed, residual, norm_weight, head)
    loss = losses.policy_loss(logits, targets, advantages).loss + 1e-3 * h.square().sum()
    d_mixed, d_residual, d_norm = torch.autograd.grad(loss, (mixed, residual, norm_weight))

    # the head's part against the same in 64 bits (the ratio is 1: minus the weighted log-probabilities' gradient)
    m64, r64, n64 = (x.detach().double().requires_grad_() for x in (mixed, residual, norm_weight))
    h64 = m64 + r64
    y64 = _Product.apply(h64 / torch.sqrt(h64.square().mean(1, keepdim=True) + 1e-6) * n64, head.dequantize().double())
    lp = torch.log_softmax(y64, 1)[torch.arange(T, device="cuda"), targets]
    (-(advantages.double() * lp).mean() + 1e-3 * h64.square().sum()).backward()
    # values near a border of two e4m3 numbers may round the other way: 2^-3 of about 1e-5 of the values, or 4e-4 of a 2-norm
    for got, want in ((logits, y64), (d_mixed, m64.grad), (d_residual, r64.grad), (d_norm, n64.grad)):
        assert float((got.detach().double() - want.detach()).norm() / want.detach().norm()) <= 4e-3

    # the block's part, from the head's gradient
    block = torch.autograd.grad((out - hidden).mean(1), [emb, *vars(w).values()], d_mixed)
    assert all(bool(x.isfinite().all()) and float(x.abs().max()) > 0 for x in block)
    grads = [block[0], d_norm, *block[1:]]
    kept = [x.clone() for x in grads]
    total = float(torch.cat([x.double().reshape(-1) for x in grads]).norm())
    n = clip.clip_grads(grads, 0.5 * total)
    assert abs(float(n) - total) <= 1e-6 * total
    for x, y in zip(grads, kept):
        assert float((x.double() - 0.5 * y.double()).abs().max()) <= 2.0 ** -22 * float(y.abs().max())
    assert abs(float(clip.grad_norm(grads)) - 0.5 * total) <= 1e-6 * total

    before = [w.w_key.detach().clone(), w.w_value.detach().clone()]
    opt = muon.MuonState([w.w_key.detach(), w.w_value.detach()])
    opt.step([grads[2], grads[3]], lr=1e-2)
    alone = muon.MuonState(before)
    alone.step([grads[2], grads[3]], lr=1e-2)
    assert torch.equal(w.w_key, before[0]) and torch.equal(w.w_value, before[1])
    # the block's kept blocks follow the updated weights
    with torch.no_grad():
        emb -= 1e-2 * grads[0]
        after, _ = ple.ple_forward(emb, hidden, w, torch.zeros(0, HC, N, device="cuda"), HP, gemm="fp8")
        fresh = ple.PleWeights(**{k: v.detach().clone() for k, v in vars(w).items()})
        assert torch.equal(after, ple.ple_forward(emb, hidden, fresh, torch.zeros(0, HC, N, device="cuda"), HP, gemm="fp8")[0])
