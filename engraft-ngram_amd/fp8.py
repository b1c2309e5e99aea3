"""Products of 8-bit floating point, with a scale for each block of 128 values:
projections kept in a quarter of their fp32 bytes, served and trained through.

* ``quantize_weight`` -- a weight ``[n, k]`` as :class:`Fp8Weight` (a scale for each
                         128 x 128 values), and its transpose for the gradient;
* ``quantize_rows``   -- activations ``[m, k]`` as :class:`Fp8Rows` (a scale for each
                         128 values of a row);
* ``product``         -- ``x @ w.T``, differentiable in ``x``;
* ``product_grad``    -- the gradient of ``x`` without autograd.

A block's values are ``q * 2^e``: ``e`` the least integer with ``max|x| <= 448 * 2^e``, q the
nearest e4m3 (4 significant bits, ties to even) of ``x * 2^-e``.  Such scales are what the
matrix cores of gfx950 take with their operands, and the values are exact in bf16.  NaN and
infinities become NaN.  The weight is frozen: its gradient is not to be had (the
``ple`` block's fp32 weights keep theirs under ``ple_forward(gemm="fp8")``).

The kernel and the order of its sums go by the number of rows: a row's result is the same bits from the same call, and
may differ in its last ones beside another number of rows.

``product`` takes the blocks of ``x`` (f32, bf16 or f16) itself; its gradient takes those of the
output's gradient, along the other axis.  f32 outputs come from exact products and fp32 sums;
16-bit ones from the fp8 matrix cores, which drop at most 2^-10 of the sum of the products' magnitudes: 1.5e-5 of an
output with normal operands, up to 5e-5 with activations that have columns far above the others (bf16 rounds by 2^-8,
f16 by 2^-11; ``out_dtype=torch.float32`` avoids it).  The reference's projections are fp32
(``engraft/replica/layers.py:594-606``)."""
from __future__ import annotations

import torch

from . import _lib


class Fp8Rows:
    """Rows in blocks: ``q`` float8_e4m3fn ``[m, k in whole blocks]`` (zeros behind k), ``scales``
    float8_e8m0fnu ``[m, blocks in fours]``."""

    __slots__ = ("q", "scales", "k")

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, k: int):
        self.q, self.scales, self.k = q, scales, k

    @property
    def shape(self) -> tuple[int, int]:
        return self.q.shape[0], self.k

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values ``[m, k]`` (exact in bf16 and f32)."""
        return _lib.autograd_ext().fp8_dequantize(self.q, self.scales, self.k, 1, _lib.dtype_code(dtype, "dtype"),
                                                  _stream(self.q))


class Fp8Weight:
    """A weight ``[n, k]`` in blocks: ``q`` float8_e4m3fn ``[n, k in whole blocks]`` (zeros behind k),
    ``scales`` float8_e8m0fnu ``[n / 128, k's blocks in fours]`` (both rounded up); ``q_t`` and ``scales_t``: the
    transpose ``[k, n]`` in the same form, the same values under the same scales, for the gradient."""

    __slots__ = ("q", "scales", "k", "q_t", "scales_t")

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, k: int, q_t: torch.Tensor | None = None,
                 scales_t: torch.Tensor | None = None):
        self.q, self.scales, self.k, self.q_t, self.scales_t = q, scales, k, q_t, scales_t

    @property
    def shape(self) -> tuple[int, int]:
        return self.q.shape[0], self.k

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values ``[n, k]`` (exact in bf16 and f32)."""
        return _lib.autograd_ext().fp8_dequantize(self.q, self.scales, self.k, 128, _lib.dtype_code(dtype, "dtype"),
                                                  _stream(self.q))


def _stream(t: torch.Tensor) -> int:
    return _lib.stream_ptr(t.device) if t.is_cuda else 0  # a host tensor is refused by the call


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """The blocks of ``x`` ``[m, k]`` f32, bf16 or f16.  Not differentiable."""
    q, scales = _lib.autograd_ext().fp8_quantize(x, _stream(x))
    return Fp8Rows(q, scales, x.shape[1])


def quantize_weight(w: torch.Tensor, *, transpose: bool = True) -> Fp8Weight:
    """The blocks of a weight ``[n, k]`` f32, bf16 or f16 of any strides; ``transpose``: with what
    the gradient needs (as many bytes again).  Not differentiable."""
    return Fp8Weight(*(lambda q, s, qt, st: (q, s, w.shape[1], qt, st))(
        *_lib.autograd_ext().fp8_quantize_weight(w, transpose, _stream(w))))


def _run(x, weight: Fp8Weight, split: int, code: int):
    """The outputs, a list of one or two 2-D tensors."""
    ext = _lib.autograd_ext()
    if isinstance(x, Fp8Rows):
        if x.k != weight.k:
            raise ValueError(f"x must have the weight's {weight.k} columns, got {x.k}")
        return ext.fp8_product(x.q, x.scales, weight.q, weight.scales, weight.k, split, code, _stream(x.q))
    return ext.fp8_linear(x, weight.q, weight.scales, weight.k, split, code, _stream(x), True)


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, split, code):
        ctx.save_for_backward(weight.q_t, weight.scales_t)
        ctx.shape, ctx.dtype, ctx.split = (x.shape[0], weight.shape[0]), x.dtype, split
        ctx.set_materialize_grads(False)
        y = _run(x, weight, split, code)
        return tuple(y) if split else y[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *d):
        if all(x is None for x in d):
            return None, None, None, None
        d_y = d[0]
        if ctx.split:  # the outputs side by side, as the weight's rows are
            rows, n = ctx.shape
            like = d[0] if d[0] is not None else d[1]
            d_y = torch.cat([like.new_zeros((rows, w)) if x is None else x for x, w in zip(d, (ctx.split, n - ctx.split))], 1)
        return _grad(d_y, *ctx.saved_tensors, ctx.shape[1], _lib.dtype_code(ctx.dtype)), None, None, None


def check_transpose(weight: Fp8Weight) -> None:
    """Raises ValueError for a weight without its transpose, which the gradient of ``x`` is a product with."""
    if weight.q_t is None or weight.scales_t is None:
        raise ValueError("the gradient of x needs the weight's transpose: fp8.quantize_weight(w, transpose=True)")
    if weight.q_t.shape[0] != weight.k:
        raise ValueError(f"the transpose of a weight {list(weight.shape)} has {weight.k} rows, got {weight.q_t.shape[0]}")


def _grad(d_y, q_t, scales_t, n, code) -> torch.Tensor:
    """``d_y @ w`` of 2-D rows from the transpose's blocks."""
    return _lib.autograd_ext().fp8_linear(d_y, q_t, scales_t, n, 0, code, _stream(d_y), False)[0]


def product(x: torch.Tensor | Fp8Rows, weight: Fp8Weight, *, out_dtype: torch.dtype | None = None,
            split: int | None = None):
    """``x @ weight.T`` for ``x`` f32, bf16 or f16 ``[..., k]`` or :class:`Fp8Rows`, as ``out_dtype`` (``x``'s; bf16
    for Fp8Rows).  ``split``: the outputs of the weight's first ``split`` rows (a multiple of 128) and of the others
    as two tensors.  Differentiable in ``x`` (a tensor) where the weight has its transpose, in reverse mode; an ``x`` with a
    forward-mode derivative is refused."""
    code = _lib.dtype_code(out_dtype if out_dtype is not None else torch.bfloat16 if isinstance(x, Fp8Rows) else x.dtype)
    if split is not None and split < 1:
        raise ValueError(f"split must be a multiple of 128 from 128 on, got {split}")
    lead = None
    if not isinstance(x, Fp8Rows) and x.dim() != 2:
        if x.dim() == 0:
            raise ValueError("x must be [..., k]")
        lead = x.shape[:-1]
        x = x.reshape(-1, x.shape[-1])
    if not isinstance(x, Fp8Rows) and x.requires_grad and torch.is_grad_enabled():
        check_transpose(weight)
        y = _Product.apply(x, weight, split or 0, code)
        y = list(y) if split else [y]
    else:
        y = _run(x, weight, split or 0, code)
    if lead is not None:
        y = [t.reshape(*lead, t.shape[-1]) for t in y]
    return tuple(y) if split else y[0]


def product_grad(d_y: torch.Tensor, weight: Fp8Weight, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The gradient of ``x`` in ``product(x, weight)`` from ``d_y`` f32, bf16 or f16 ``[..., n]``: ``d_y @ weight``,
    as ``dtype`` (``d_y``'s)."""
    check_transpose(weight)
    if d_y.dim() == 0:
        raise ValueError("d_y must be [..., n]")
    code = _lib.dtype_code(dtype if dtype is not None else d_y.dtype, "dtype")
    rows = d_y if d_y.dim() == 2 else d_y.reshape(-1, d_y.shape[-1])
    d_x = _grad(rows, weight.q_t, weight.scales_t, weight.shape[0], code)
    return d_x if d_y.dim() == 2 else d_x.reshape(*d_y.shape[:-1], weight.k)
