"""The norm of all gradients of a step, and their clipping: what stands between the gradients
(of table rows, of the PLE block's norms and projections) and the updates of ``muon`` or
``descent``.

* ``grad_norm``  -- the 2-norm of a list of tensors as one vector;
* ``clip_grads`` -- the same, with the tensors scaled to a norm of at most ``max_norm``.

Squares are added in 64 bits, in an order that the sizes alone decide, so a norm is the same
bits every time; nothing is synchronised or copied to the device.  Neither is differentiable."""
from __future__ import annotations

import torch

from . import _lib


def _stream(t: torch.Tensor) -> int:
    return _lib.stream_ptr(t.device) if t.is_cuda else 0  # a host tensor is refused by the call


def _list(grads) -> list:
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        raise ValueError("no gradients")
    return grads


def grad_norm(grads) -> torch.Tensor:
    """0-d f32 on the GPU: the 2-norm of ``grads`` (tensors f32, bf16 or f16 on one GPU, without gaps or rows of unit
    stride) as one vector."""
    grads = _list(grads)
    return _lib.autograd_ext().clip(grads, None, 0.0, _stream(grads[0]))


def clip_grads(grads, max_norm: float, *, out=None) -> torch.Tensor:
    """:func:`grad_norm`'s value N, with every gradient times ``max_norm / N`` where ``N > max_norm``, in place or as
    ``out`` (tensors of the gradients' shapes, f32, bf16 or f16: all are written, clipped or not).  A norm that is not finite
    leaves the values as they are.  A gradient given twice (or two that share a value) is refused, as are outputs that
    overlap anything else."""
    grads = _list(grads)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    return _lib.autograd_ext().clip(grads, grads if out is None else _list(out), max_norm, _stream(grads[0]))
