"""Orthogonalised weight updates: the optimizer of the PLE block's projection
weights, whose gradients ``ple.ple_forward``'s backward gives (table rows keep
``DescentState``'s Adam).

For each matrix on its own: momentum, then the update's singular values are
driven to about 1 by Newton-Schulz products (a quintic polynomial of the matrix,
on the fp16 matrix cores), then a step:

    m = momentum m + g
    u = g + momentum m  (nesterov)  or  m
    X = u / (|u|_F + eps);   steps times:  X = a X + (b A + c A^2) X,  A = X X^T
    w = (1 - lr weight_decay) w - lr sqrt(max(1, rows / cols)) X

* ``muon_step``     -- one step of given weights, gradients and momenta;
* ``MuonState``     -- the same with the momenta kept;
* ``orthogonalize`` -- X alone.

Products: a step takes fp32 accuracy whatever the weights' type (operands as two fp16
planes, 22 bits, three products: ``products="fp16x3"``).  ``products="fp16"`` is one
product of 11-bit operands, in half the time or less: X is then off by 1.1e-3 of itself,
which moves some bf16 weights by one unit in the last place.  ``orthogonalize`` takes it
by itself for a bf16 matrix, whose X is rounded to 8 bits in the end."""
from __future__ import annotations

import torch

from . import _lib

QUINTIC = (3.4445, -4.7750, 2.0315)
_PLANES = {None: 0, "fp16x3": 2, "fp16": 1}


def _coefficients(coefficients, steps: int) -> list[float]:
    """``steps`` rows (a, b, c), flat: one triple for all steps, or one each."""
    rows = [tuple(coefficients)] * steps if coefficients and not isinstance(coefficients[0], (tuple, list)) \
        else [tuple(c) for c in coefficients]
    if steps < 1 or len(rows) != steps or any(len(c) != 3 for c in rows):
        raise ValueError(f"coefficients must be one (a, b, c) or {steps} of them, got {coefficients!r}")
    return [x for c in rows for x in c]


def _run(params, grads, momenta, steps, coefficients, products, *args):
    if products not in _PLANES:
        raise ValueError(f"products must be one of {tuple(_PLANES)}, got {products!r}")
    stream = _lib.stream_ptr(params[0].device) if params and params[0].is_cuda else 0
    _lib.autograd_ext().muon(params, grads, momenta, _coefficients(coefficients, steps), steps, _PLANES[products], *args,
                             stream)


def muon_step(params, grads, momenta, *, lr: float, weight_decay: float = 0.0, momentum: float = 0.95,
              nesterov: bool = True, steps: int = 5, coefficients=QUINTIC, eps: float = 1e-7,
              products: str | None = None) -> None:
    """One step of ``params`` (a list of f32, bf16 or f16 ``[rows, cols]`` or
    ``[count, rows, cols]``, each matrix an update of its own), in place, with
    ``momenta`` (f32, the same shapes), in place, from ``grads``.  Any strides, one device;
    matrices of one shape, type and strides share their launches.  Weights and momenta must not
    overlap themselves, each other (a weight given twice is refused) or the gradients, but a weight may
    be over its own gradient.  A step is whole or not at all: where a matrix is refused, or there is no
    memory for the workspace, nothing is stepped.  ``coefficients``: one (a, b, c) for every
    Newton-Schulz step, or one each.  ``products``: "fp16x3" (None: the same) or "fp16"."""
    _run(list(params), list(grads), list(momenta), steps, coefficients, products, nesterov, momentum, eps,
         1.0 - lr * weight_decay, lr, True)


def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients=QUINTIC, eps: float = 1e-7,
                  out: torch.Tensor | None = None, products: str | None = None) -> torch.Tensor:
    """``x`` (f32, bf16 or f16 ``[rows, cols]`` or ``[count, rows, cols]``) with every matrix's
    singular values driven to about 1, in ``x``'s type.  ``out``: where it is written (``x`` for in place).
    ``products`` None: "fp16" for bf16, "fp16x3" otherwise."""
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _run([out], [x], [], steps, coefficients, products, False, 0.0, eps, 0.0, 0.0, False)
    return out


class MuonState:
    """Weights and their momenta.  ``params``: ``PleWeights.w_key`` as ``[streams, n, n]``,
    ``w_value``, or other 2-D weights; ``momenta``: f32 tensors to go on from (zeros otherwise)."""

    def __init__(self, params, momenta=None, *, momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
                 coefficients=QUINTIC, eps: float = 1e-7, products: str | None = None):
        self.params = list(params)
        if any(not w.is_cuda for w in self.params):
            raise ValueError("params must be on the GPU")
        self.momenta = [torch.zeros(w.shape, dtype=torch.float32, device=w.device) for w in self.params] \
            if momenta is None else list(momenta)
        self._options = dict(momentum=momentum, nesterov=nesterov, steps=steps, coefficients=coefficients, eps=eps,
                             products=products)
        self.step_count = 0

    def step(self, grads, *, lr: float, weight_decay: float = 0.0) -> None:
        """One step of every weight from its gradient."""
        muon_step(self.params, grads, self.momenta, lr=lr, weight_decay=weight_decay, **self._options)
        self.step_count += 1  # only once the step is on its way
