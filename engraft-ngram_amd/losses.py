"""Losses of next-token logits, with the gradient of the logits: what a
descent's ``d_out`` comes from when the rows or the PLE block's weights are
trained on answers that are preferred or rewarded.  The reference policy of
both losses is the same model without the overlay.

* ``token_logprobs``        -- the targets' log-probabilities (scores of the
                               reference policy or of sampled answers);
* ``policy_loss``           -- the clipped policy loss with a KL term;
* ``preference_loss``       -- the loss of paired log ratios of whole answers;
* ``policy_loss_grad``, ``preference_loss_grad`` -- the same with the gradient
  of the logits in one call, without autograd.

``logits`` are ``[n, vocab]`` f32, bf16 or f16 on the GPU, one row a position
(a packed bin's prefix positions, ``pack.Packed``), rows any stride of at least
``vocab`` apart and unit stride within a row; ``targets`` int64 or int32
``[n]``.  A row whose target is negative (a prompt's position, a packed
fragment's boundary) is left out: its logits are not read, its gradient is
zero.  A target outside the vocabulary gives NaN.  Gradients have the logits'
type; everything else is f32 (sums over rows and sequences are kept in 64
bits).  The reference trains on a teacher's distribution instead
(``engraft/replica/distill.py:283-325``)."""
from __future__ import annotations

import dataclasses

import torch

from . import _lib

_REDUCTIONS = {"sum": 0, "token": 1, "sequence": 2}  # eg_reduction


@dataclasses.dataclass
class PolicyLoss:
    """``loss``: differentiable in the logits (from :func:`policy_loss`); ``kl``
    and ``clip_fraction``: the weighted KL term and the weighted share of rows
    whose clipped ratio is the smaller product; all three 0-d f32.
    ``logprobs`` f32 ``[n]``: the targets', 0 in rows that are left out."""

    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor
    logprobs: torch.Tensor


@dataclasses.dataclass
class PreferenceLoss:
    """``loss``: 0-d f32, differentiable in the logits (from
    :func:`preference_loss`); ``margins`` f32 ``[pairs]``: beta times the
    difference of the pair's log ratios (the chosen answer wins above 0);
    ``sequence_logprobs`` f32 ``[2 * pairs]`` and ``logprobs`` f32 ``[n]``."""

    loss: torch.Tensor
    margins: torch.Tensor
    sequence_logprobs: torch.Tensor
    logprobs: torch.Tensor


def _stream(t: torch.Tensor) -> int:
    return _lib.stream_ptr(t.device) if t.is_cuda else 0  # a host tensor is refused by the call


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """f32 ``[n]``: ``log_softmax(logits / temperature)`` at the targets, 0 where a
    target is negative.  Not differentiable."""
    return _lib.autograd_ext().token_logprobs(logits, targets, temperature, _stream(logits))


def _policy(logits, targets, advantages, old_logprobs, ref_logprobs, segment_ids, n_segments, clip, kl_coef,
            temperature, reduction, grad=False, out=None, grad_scale=1.0):
    """``(state, loss, kl, clip_fraction, logprobs, d_logits)`` of one ``eg_policy_loss`` call."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    if ref_logprobs is None and kl_coef != 0.0:
        raise ValueError("the KL term needs ref_logprobs")
    if reduction == "sequence" and (segment_ids is None or n_segments is None):
        raise ValueError("reduction='sequence' needs segment_ids and n_segments")
    return _lib.autograd_ext().policy(logits, targets, advantages, old_logprobs, ref_logprobs, segment_ids,
                                      n_segments or 0, clip[0], clip[1], kl_coef, temperature, _REDUCTIONS[reduction],
                                      grad, out, grad_scale, _stream(logits))


def _preference(logits, targets, segment_ids, ref_logprobs, beta, label_smoothing, temperature, grad=False, out=None,
                grad_scale=1.0):
    """``(state, loss, margins, sequence_logprobs, logprobs, d_logits)`` of one ``eg_preference_loss`` call."""
    return _lib.autograd_ext().preference(logits, targets, segment_ids, ref_logprobs, beta, label_smoothing, temperature,
                                          grad, out, grad_scale, _stream(logits))


def _logits_grad(ctx, upstream):
    """The gradient pass from a loss's saved state, times the loss's own gradient."""
    logits, targets, state = ctx.saved_tensors
    return _lib.autograd_ext().logits_grad(logits, targets, ctx.temperature, state, upstream, _stream(logits))


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, *args):
        state, loss, kl, clipped, lp, _ = _policy(logits, targets, *args)
        ctx.save_for_backward(logits, targets, state)
        ctx.temperature = args[7]
        ctx.mark_non_differentiable(kl, clipped, lp)
        return loss, kl, clipped, lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss, *_):
        return (_logits_grad(ctx, d_loss),) + (None,) * 10


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, *args):
        state, loss, margins, seqs, lp, _ = _preference(logits, targets, *args)
        ctx.save_for_backward(logits, targets, state)
        ctx.temperature = args[4]
        ctx.mark_non_differentiable(margins, seqs, lp)
        return loss, margins, seqs, lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss, *_):
        return (_logits_grad(ctx, d_loss),) + (None,) * 6


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor,
                old_logprobs: torch.Tensor | None = None, *, ref_logprobs: torch.Tensor | None = None,
                segment_ids: torch.Tensor | None = None, n_segments: int | None = None, clip=(0.2, 0.2),
                kl_coef: float = 0.0, temperature: float = 1.0, reduction: str = "token") -> PolicyLoss:
    """The clipped policy loss with a KL term, differentiable in the logits.

    With ``lp`` the targets' log-probabilities under ``logits / temperature``,
    ``r = exp(lp - old_logprobs)``, ``A = advantages`` and ``d = ref_logprobs - lp``:

        sum_i w_i (-min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (e^d - d - 1))

    ``old_logprobs`` None: the policy's own, a ratio of 1 whose gradient stays.
    Where the two products are equal the gradient is the first's.  Weights by
    ``reduction``: ``"sum"`` 1; ``"token"`` 1 / the rows that have a target;
    ``"sequence"`` 1 / (segments that have such a row * the segment's), with
    ``segment_ids`` (``[n]``, any order; a value outside ``[0, n_segments)`` gives
    its row no weight).  No gradient flows into the other arguments; the
    logits must not change before the backward."""
    loss, kl, clipped, lp = _PolicyLoss.apply(logits, targets, advantages, old_logprobs, ref_logprobs, segment_ids,
                                              n_segments, clip, kl_coef, temperature, reduction)
    return PolicyLoss(loss, kl, clipped, lp)


def policy_loss_grad(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor,
                     old_logprobs: torch.Tensor | None = None, *, ref_logprobs: torch.Tensor | None = None,
                     segment_ids: torch.Tensor | None = None, n_segments: int | None = None, clip=(0.2, 0.2),
                     kl_coef: float = 0.0, temperature: float = 1.0, reduction: str = "token",
                     grad_scale: float = 1.0, out: torch.Tensor | None = None) -> tuple[PolicyLoss, torch.Tensor]:
    """:func:`policy_loss` and the gradient of ``grad_scale`` times it, as
    ``(PolicyLoss, d_logits)`` without autograd.  ``out``: where the gradient is
    written (the logits themselves for in place; over part of them, or over
    another argument, is refused)."""
    _, loss, kl, clipped, lp, d = _policy(logits, targets, advantages, old_logprobs, ref_logprobs, segment_ids, n_segments,
                                          clip, kl_coef, temperature, reduction, True, out, grad_scale)
    return PolicyLoss(loss, kl, clipped, lp), d


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, segment_ids: torch.Tensor,
                    ref_logprobs: torch.Tensor, *, beta: float = 0.1, label_smoothing: float = 0.0,
                    temperature: float = 1.0) -> PreferenceLoss:
    """The preference loss of paired log ratios, differentiable in the logits.

    ``segment_ids`` ``[n]``, not decreasing (``Packed.segment_ids``): segment ``2 p``
    is pair ``p``'s chosen answer, ``2 p + 1`` its rejected one; ids past the pairs
    belong to none.  ``ref_logprobs`` ``[2 * pairs]``: the reference policy's sums.
    With ``s_k`` segment ``k``'s sum of log-probabilities and
    ``h_p = beta ((s_2p - ref_2p) - (s_2p+1 - ref_2p+1))``:

        mean_p(-(1 - label_smoothing) log sigma(h_p) - label_smoothing log sigma(-h_p))

    Segments out of order give NaN (sums, margins, loss, gradient).  The logits must not change before the
    backward."""
    return PreferenceLoss(*_PreferenceLoss.apply(logits, targets, segment_ids, ref_logprobs, beta, label_smoothing,
                                                 temperature))


def preference_loss_grad(logits: torch.Tensor, targets: torch.Tensor, segment_ids: torch.Tensor,
                         ref_logprobs: torch.Tensor, *, beta: float = 0.1, label_smoothing: float = 0.0,
                         temperature: float = 1.0, grad_scale: float = 1.0,
                         out: torch.Tensor | None = None) -> tuple[PreferenceLoss, torch.Tensor]:
    """:func:`preference_loss` and the gradient of ``grad_scale`` times it, as
    ``(PreferenceLoss, d_logits)`` without autograd.  ``out``: where the gradient is
    written (the logits themselves for in place; over part of them, or over
    another argument, is refused)."""
    _, loss, margins, seqs, lp, d = _preference(logits, targets, segment_ids, ref_logprobs, beta, label_smoothing,
                                                temperature, True, out, grad_scale)
    return PreferenceLoss(loss, margins, seqs, lp), d
