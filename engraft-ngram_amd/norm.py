"""The residual's addition and the RMS norm of the sum: what stands between the PLE block's
output (or any layer's) and the projections behind it.

    h = x + residual            (rounded to the residual's type)
    y = h weight / sqrt(mean(h^2) + eps)

* ``add_rms_norm``, ``rms_norm`` -- ``(y, h)``, and ``y`` without a residual, differentiable;
                                    with ``out_dtype="fp8"`` y as ``fp8.Fp8Rows``;
* ``add_rms_norm_stats``, ``add_rms_norm_grad`` -- the same without autograd;
* ``normed_product``             -- ``fp8.product`` of the normed rows, the norm writing them in 8
                                    bits, differentiable.

``x`` is f32, bf16 or f16 ``[..., d]``, d up to 20,480; the residual of x's type or f32;
the weight f32, bf16 or f16 ``[d]`` or None (1).  Eight squares are added in 32 bits (in 64
where they leave its range), their sums and the root in 64, gradients in 32 and in reverse mode (inputs with a forward-mode derivative are refused); rows in 8 bits round as the exact ones do, but for one value in millions.  The reference's rms norm is a torch expression
(``engraft/lens.py:282-287``), its additions are apart."""
from __future__ import annotations

import torch

from . import _lib, fp8


def _stream(t: torch.Tensor) -> int:
    return _lib.stream_ptr(t.device) if t.is_cuda else 0  # a host tensor is refused by the call


def _flat(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None or t.dim() == 2:
        return t
    if t.dim() == 0:
        raise ValueError("rows [..., d] expected, got a number")
    return t.reshape(-1, t.shape[-1])


def _code(out_dtype, x: torch.Tensor) -> int:
    return -1 if out_dtype == "fp8" else _lib.dtype_code(x.dtype if out_dtype is None else out_dtype)


def _forward(x, residual, weight, eps, code, stats, differentiable=True):
    """``(y, h, rstd)`` of 2-D rows, y Fp8Rows for code -1."""
    if not eps >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    y, scales, h, rstd = _lib.autograd_ext().norm(x, residual, weight, eps, code, stats, _stream(x), differentiable)
    return (fp8.Fp8Rows(y, scales, x.shape[1]) if code < 0 else y), h, rstd


def add_rms_norm_stats(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, *, eps: float = 1e-6,
                       out_dtype: torch.dtype | str | None = None):
    """``(y, h, rstd)`` without autograd: y of ``out_dtype`` (x's; "fp8": ``Fp8Rows``), h in the residual's type (x itself
    without one), rstd f32 ``[rows]`` for :func:`add_rms_norm_grad`.  Rows ``[n, d]``."""
    return _forward(x, residual, weight, eps, _code(out_dtype, x), True, False)


def add_rms_norm_grad(d_y: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None, *,
                      d_residual: torch.Tensor | None = None, dtype: torch.dtype | None = None):
    """``(d_h, d_weight)`` from the gradient of y, and of h (``d_residual``, h's type): d_h, that of x and of the residual alike,
    of ``dtype`` (h's), d_weight of the weight's type (None without one).  Rows ``[n, d]``."""
    d_h, _, d_w = _lib.autograd_ext().norm_grad(d_y, h, rstd, weight, d_residual,
                                                _lib.dtype_code(h.dtype if dtype is None else dtype, "dtype"), -1,
                                                weight is not None, _stream(h))
    return d_h, d_w


def _norm_backward(ctx, d_y, d_h):
    """The gradients of x, the residual and the weight; d_y the normed rows' (None: none)."""
    h, rstd, weight = ctx.saved_tensors[:3]
    need_x, need_r, need_w = ctx.needs_input_grad[:3]
    x_dtype, r_dtype = ctx.dtypes
    if d_h is not None and d_h.dtype != h.dtype:
        d_h = d_h.to(h.dtype)
    if d_y is None:  # the loss reaches h alone
        d_w = torch.zeros_like(weight) if need_w else None
        return (d_h.to(x_dtype) if need_x else None), (d_h.to(r_dtype) if need_r else None), d_w
    first = x_dtype if need_x or not need_r else r_dtype
    second = r_dtype if need_x and need_r and r_dtype != x_dtype else None
    d_x, d_r, d_w = _lib.autograd_ext().norm_grad(d_y, h, rstd, weight, d_h, _lib.dtype_code(first),
                                                  -1 if second is None else _lib.dtype_code(second), need_w, _stream(h))
    if need_r and second is None:
        d_r = d_x.clone() if need_x else d_x  # a gradient each: one may be added to in place
    return (d_x if need_x else None), (d_r if need_r else None), d_w


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, code):
        y, h, rstd = _forward(x, residual, weight, eps, code, True)
        ctx.save_for_backward(h, rstd, weight)
        ctx.dtypes = (x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_h=None):
        if d_y is None and d_h is None:
            return None, None, None, None, None
        return (*_norm_backward(ctx, d_y, d_h), None, None)


def _differentiates(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                 out_dtype: torch.dtype | str | None = None):
    """``(y, h)``: h = x + residual in the residual's type, y its RMS norm times the weight as ``out_dtype`` (x's).
    Differentiable in x, the residual and the weight; ``out_dtype="fp8"`` gives y as ``fp8.Fp8Rows``, which has no gradient
    (:func:`normed_product` has), and refuses inputs that require one."""
    if residual.shape != x.shape:
        raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
    return _call(x, residual, weight, eps, out_dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, eps: float = 1e-6,
             out_dtype: torch.dtype | str | None = None):
    """:func:`add_rms_norm` of ``x`` alone: y."""
    return _call(x, None, weight, eps, out_dtype)


def _call(x, residual, weight, eps, out_dtype):
    code = _code(out_dtype, x)
    x2, r2 = _flat(x), _flat(residual)
    if _differentiates(x, residual, weight):
        if code < 0:
            raise ValueError("rows in 8 bits have no gradient: normed_product, or no_grad")
        out = _AddRmsNorm.apply(x2, r2, weight, eps, code)
        y, h = (out, None) if residual is None else out
    else:
        y, h, _ = _forward(x2, r2, weight, eps, code, False)
    if code >= 0:
        y = y.reshape(x.shape)
    return y if residual is None else (y, h.reshape(x.shape))


class _NormedProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, norm_weight, weight, eps, code):
        rows, h, rstd = _forward(x, residual, norm_weight, eps, -1, True)
        ctx.save_for_backward(h, rstd, norm_weight, weight.q_t, weight.scales_t)
        ctx.n = weight.shape[0]
        ctx.dtypes = (x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        y = fp8._run(rows, weight, 0, code)[0]
        return y if residual is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_h=None):
        if d_y is None and d_h is None:
            return None, None, None, None, None, None
        # fp32: the norm's gradients are sums over a row and over all rows of it
        d_rows = None if d_y is None else fp8._grad(d_y, *ctx.saved_tensors[3:], ctx.n, 0)
        return (*_norm_backward(ctx, d_rows, d_h), None, None, None)


def normed_product(x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor | None, weight: fp8.Fp8Weight,
                   *, eps: float = 1e-6, out_dtype: torch.dtype | None = None):
    """``(fp8.product(rows, weight), h)`` with ``rows, h`` those of :func:`add_rms_norm` in 8 bits; without a residual
    the product alone.  ``out_dtype`` None: x's.  Differentiable in x, the residual and the norm's weight: the rounding to 8 bits
    passes its gradient on."""
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
    code = _lib.dtype_code(x.dtype if out_dtype is None else out_dtype)
    x2, r2 = _flat(x), _flat(residual)
    if x2.shape[1] != weight.k:
        raise ValueError(f"x must have the weight's {weight.k} columns, got {list(x.shape)}")
    if _differentiates(x, residual, norm_weight):
        fp8.check_transpose(weight)
        out = _NormedProduct.apply(x2, r2, norm_weight, weight, eps, code)
        y, h = (out, None) if residual is None else out
    else:
        rows, h, _ = _forward(x2, r2, norm_weight, eps, -1, False)
        y = fp8._run(rows, weight, 0, code)[0]
    y = y.reshape(*x.shape[:-1], y.shape[-1])
    return y if residual is None else (y, h.reshape(x.shape))
