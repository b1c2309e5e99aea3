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

import ctypes
import dataclasses

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # eg_dtype
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


def _integers(x: torch.Tensor, n: int, name: str, dev) -> tuple[torch.Tensor, int]:
    """``x`` as contiguous int64 or int32 ``[n]`` on ``dev``, and whether it is int32."""
    if x.device != dev or x.dim() != 1 or x.shape[0] != n:
        raise ValueError(f"{name} must be [{n}] on {dev}, got {list(x.shape)} on {x.device}")
    if x.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32, got {x.dtype}")
    return (x if x.is_contiguous() else x.contiguous()), int(x.dtype == torch.int32)


def _floats(x: torch.Tensor, n: int, name: str, dev) -> torch.Tensor:
    """``x`` as contiguous f32 ``[n]`` on ``dev``."""
    if x.device != dev or x.dim() != 1 or x.shape[0] != n or not x.is_floating_point():
        raise ValueError(f"{name} must be floating [{n}] on {dev}, got {x.dtype} {list(x.shape)} on {x.device}")
    x = x if x.dtype == torch.float32 else x.float()
    return x if x.is_contiguous() else x.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _c_logits(logits: torch.Tensor, targets: torch.Tensor, temperature: float) -> tuple[_lib.EgLogits, torch.Tensor]:
    if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError(f"logits must be f32, bf16 or f16 [n, vocab] on the GPU, got {logits.dtype} "
                         f"{list(logits.shape)} on {logits.device}")
    n, v = logits.shape
    if v > 1 and logits.stride(1) != 1:
        raise ValueError(f"logits must have unit stride within a row, got strides {tuple(logits.stride())}")
    targets, i32 = _integers(targets, n, "targets", logits.device)
    return _lib.EgLogits(_lib.ptr(logits) if n else None, _DTYPES[logits.dtype], i32, n, v, _row_stride(logits),
                         _lib.ptr(targets) if n else None, float(temperature)), targets


def _scratch(c: _lib.EgLogits, n_segments: int, with_state: bool, dev) -> tuple[torch.Tensor, int, int]:
    """One buffer of a call: its rows' state (12 bytes each), then the workspace;
    the workspace's offset and size."""
    size = _lib.load().eg_loss_workspace_size(c.n, c.v, c.dtype, n_segments)
    if size < 0:
        raise ValueError(f"a loss of {c.n} rows, a vocabulary of {c.v} and {n_segments} segments")
    first = (12 * c.n + 15) // 16 * 16 if with_state else 0
    return torch.empty(first + size, dtype=torch.uint8, device=dev), first, size


def _gradient(logits: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or \
            (out.shape[1] > 1 and out.stride(1) != 1):
        raise ValueError(f"out must be {logits.dtype} {list(logits.shape)} on {logits.device} with unit stride within "
                         "a row")
    return out


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """f32 ``[n]``: ``log_softmax(logits / temperature)`` at the targets, 0 where a
    target is negative.  Not differentiable."""
    c, targets = _c_logits(logits, targets, temperature)
    dev = logits.device
    lp = torch.empty(c.n, dtype=torch.float32, device=dev)
    ws, _, size = _scratch(c, 0, False, dev)
    _lib.call("eg_token_logprobs", ctypes.byref(c), _lib.ptr(lp), _lib.ptr(ws), size, _lib.stream_ptr(dev))
    return lp


def _policy(logits, targets, advantages, old_logprobs, ref_logprobs, segment_ids, n_segments, clip, kl_coef,
            temperature, reduction, d_logits, grad_scale):
    """``(c_logits, targets, scratch, sums, logprobs)`` of one ``eg_policy_loss`` call."""
    c, targets = _c_logits(logits, targets, temperature)
    dev, n = logits.device, c.n
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    p = _lib.EgPolicy()
    advantages = _floats(advantages, n, "advantages", dev)
    p.advantages = _lib.ptr(advantages)
    if old_logprobs is not None:
        old_logprobs = _floats(old_logprobs, n, "old_logprobs", dev)
        p.old_logprobs = _lib.ptr(old_logprobs)
    if ref_logprobs is not None:
        ref_logprobs = _floats(ref_logprobs, n, "ref_logprobs", dev)
        p.ref_logprobs = _lib.ptr(ref_logprobs)
    elif kl_coef != 0.0:
        raise ValueError("the KL term needs ref_logprobs")
    p.reduction = _REDUCTIONS[reduction]
    count = 0
    if reduction == "sequence":
        if segment_ids is None or n_segments is None:
            raise ValueError("reduction='sequence' needs segment_ids and n_segments")
        segment_ids, p.segment_ids_i32 = _integers(segment_ids, n, "segment_ids", dev)
        p.segment_ids, p.n_segments = _lib.ptr(segment_ids), int(n_segments)
        count = max(p.n_segments, 0)
    p.clip_low, p.clip_high, p.kl_coef = float(clip[0]), float(clip[1]), float(kl_coef)
    scratch, first, size = _scratch(c, count, True, dev)
    sums = torch.empty(3, dtype=torch.float32, device=dev)
    lp = torch.empty(n, dtype=torch.float32, device=dev)
    at = _lib.ptr(scratch)
    _lib.call("eg_policy_loss", ctypes.byref(c), ctypes.byref(p), _lib.ptr(lp), _lib.ptr(sums), at,
              _lib.ptr(d_logits) if d_logits is not None and n else None,
              _row_stride(d_logits) if d_logits is not None else 0, float(grad_scale), at + first, size,
              _lib.stream_ptr(dev))
    return c, targets, scratch, sums, lp


def _preference(logits, targets, segment_ids, ref_logprobs, beta, label_smoothing, temperature, d_logits, grad_scale):
    """``(c_logits, targets, scratch, loss, margins, sequence_logprobs, logprobs)`` of one
    ``eg_preference_loss`` call."""
    c, targets = _c_logits(logits, targets, temperature)
    dev, n = logits.device, c.n
    if ref_logprobs.dim() != 1 or ref_logprobs.shape[0] < 2 or ref_logprobs.shape[0] % 2:
        raise ValueError(f"ref_logprobs must be [2 * pairs] (chosen, rejected, ...), got {list(ref_logprobs.shape)}")
    count = ref_logprobs.shape[0]
    ref_logprobs = _floats(ref_logprobs, count, "ref_logprobs", dev)
    segment_ids, i32 = _integers(segment_ids, n, "segment_ids", dev)
    p = _lib.EgPreference(_lib.ptr(segment_ids), _lib.ptr(ref_logprobs), count // 2, i32, float(beta),
                          float(label_smoothing))
    scratch, first, size = _scratch(c, count, True, dev)
    sums = torch.empty(1 + count // 2 + count, dtype=torch.float32, device=dev)
    lp = torch.empty(n, dtype=torch.float32, device=dev)
    at, to = _lib.ptr(scratch), _lib.ptr(sums)
    _lib.call("eg_preference_loss", ctypes.byref(c), ctypes.byref(p), _lib.ptr(lp), to + 4 * (1 + count // 2), to + 4,
              to, at, _lib.ptr(d_logits) if d_logits is not None and n else None,
              _row_stride(d_logits) if d_logits is not None else 0, float(grad_scale), at + first, size,
              _lib.stream_ptr(dev))
    return c, targets, scratch, sums[0], sums[1:1 + count // 2], sums[1 + count // 2:], lp


def _logits_grad(ctx, upstream):
    """The gradient pass from a loss's saved state, times the loss's own gradient."""
    logits, targets, scratch = ctx.saved_tensors
    c, _ = _c_logits(logits, targets, ctx.temperature)
    d = _gradient(logits, None)
    up = upstream if upstream.dtype == torch.float32 else upstream.float()
    _lib.call("eg_logits_grad", ctypes.byref(c), _lib.ptr(scratch), _lib.ptr(up), 1.0,
              _lib.ptr(d) if c.n else None, _row_stride(d), _lib.stream_ptr(logits.device))
    return d


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, *args):
        _, targets, scratch, sums, lp = _policy(logits, targets, *args, None, 1.0)
        ctx.save_for_backward(logits, targets, scratch)
        ctx.temperature = args[7]
        loss, kl, clipped = sums[0].clone(), sums[1], sums[2]
        ctx.mark_non_differentiable(kl, clipped, lp)
        return loss, kl, clipped, lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss, *_):
        return (_logits_grad(ctx, d_loss),) + (None,) * 10


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, *args):
        _, targets, scratch, loss, margins, seqs, lp = _preference(logits, targets, *args, None, 1.0)
        ctx.save_for_backward(logits, targets, scratch)
        ctx.temperature = args[4]
        loss = loss.clone()
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
    written (the logits themselves for in place)."""
    with torch.no_grad():
        d = _gradient(logits, out)
        _, _, _, sums, lp = _policy(logits, targets, advantages, old_logprobs, ref_logprobs, segment_ids, n_segments,
                                    clip, kl_coef, temperature, reduction, d, grad_scale)
    return PolicyLoss(sums[0], sums[1], sums[2], lp), d


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

    Segments out of order give NaN.  The logits must not change before the
    backward."""
    return PreferenceLoss(*_PreferenceLoss.apply(logits, targets, segment_ids, ref_logprobs, beta, label_smoothing,
                                                 temperature))


def preference_loss_grad(logits: torch.Tensor, targets: torch.Tensor, segment_ids: torch.Tensor,
                         ref_logprobs: torch.Tensor, *, beta: float = 0.1, label_smoothing: float = 0.0,
                         temperature: float = 1.0, grad_scale: float = 1.0,
                         out: torch.Tensor | None = None) -> tuple[PreferenceLoss, torch.Tensor]:
    """:func:`preference_loss` and the gradient of ``grad_scale`` times it, as
    ``(PreferenceLoss, d_logits)`` without autograd.  ``out``: where the gradient is
    written (the logits themselves for in place)."""
    with torch.no_grad():
        d = _gradient(logits, out)
        _, _, _, loss, margins, seqs, lp = _preference(logits, targets, segment_ids, ref_logprobs, beta,
                                                       label_smoothing, temperature, d, grad_scale)
    return PreferenceLoss(loss, margins, seqs, lp), d
