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

Products: fp32 weights take fp32 accuracy (operands as two fp16 planes, 22 bits,
three products), bf16 and f16 weights one product of 11-bit operands, whose
error stays below the weight's own rounding; ``products`` overrides."""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # eg_dtype
QUINTIC = (3.4445, -4.7750, 2.0315)
_PLANES = {"fp16x3": 2, "fp16": 1}


class _Workspace:
    """Grow-only device workspace, one per (device, stream): calls on one stream run in
    order and may share it, calls on different streams never do.  A captured call takes a
    buffer of its own from the graph's pool: a kept one could be replaced while the graph lives."""

    def __init__(self):
        self._buf: dict[tuple[torch.device, int], torch.Tensor] = {}

    def get(self, need: int, dev: torch.device) -> torch.Tensor:
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                return torch.empty(need, dtype=torch.uint8, device=dev)
        key = (dev, _lib.stream_ptr(dev))
        buf = self._buf.get(key)
        if buf is None or buf.numel() < need:
            buf = torch.empty(need, dtype=torch.uint8, device=dev)
            self._buf[key] = buf
        return buf


_WS = _Workspace()


def _coefficients(coefficients, steps: int):
    """``steps`` rows (a, b, c) as a host array: one triple for all steps, or one each."""
    rows = [tuple(coefficients)] * steps if coefficients and not isinstance(coefficients[0], (tuple, list)) \
        else [tuple(c) for c in coefficients]
    if steps < 1 or len(rows) != steps or any(len(c) != 3 for c in rows):
        raise ValueError(f"coefficients must be one (a, b, c) or {steps} of them, got {coefficients!r}")
    return (ctypes.c_float * (3 * steps))(*(x for c in rows for x in c))


def _planes(products: str | None, dtype: torch.dtype) -> int:
    if products is None:
        return 2 if dtype == torch.float32 else 1
    if products not in _PLANES:
        raise ValueError(f"products must be one of {tuple(_PLANES)}, got {products!r}")
    return _PLANES[products]


def _check(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    if t.dim() not in (2, 3) or t.dtype not in _DTYPES or not t.is_cuda:
        raise ValueError(f"{name} must be f32, bf16 or f16 [rows, cols] or [count, rows, cols] on the GPU, got "
                         f"{t.dtype} {list(t.shape)} on {t.device}")
    if like is not None and (t.shape != like.shape or t.device != like.device):
        raise ValueError(f"{name} must be {list(like.shape)} on {like.device} like its weight, got {list(t.shape)} on "
                         f"{t.device}")


def _writable(t: torch.Tensor, name: str) -> None:
    if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} is written and must not be expanded, got strides {tuple(t.stride())}")


def _places(t: torch.Tensor) -> list[int]:
    """Device address of every matrix of ``t``."""
    if t.dim() == 2:
        return [t.data_ptr()]
    step = t.stride(0) * t.element_size()
    return [t.data_ptr() + i * step for i in range(t.shape[0])]


def _run(params, grads, momenta, planes, table, steps, *, momentum, nesterov, eps, keep, rate_of):
    """One ``eg_muon_step`` per group of matrices of the same shape, types and strides."""
    groups: dict = {}
    for i, (w, g) in enumerate(zip(params, grads)):
        if w.numel() == 0:
            continue
        m = momenta[i] if momenta is not None else None
        key = (w.device, w.shape[-2:], w.dtype, g.dtype, w.stride()[-2:], g.stride()[-2:],
               m.stride()[-2:] if m is not None else None)
        groups.setdefault(key, []).append((w, g, m))
    for (dev, shape, wt, gt, ws, gs, ms), members in groups.items():
        at = [[], [], []]
        for trio in members:
            for to, t in zip(at, trio):
                if t is not None:
                    to.extend(_places(t))
        count = len(at[0])
        arrays = [(ctypes.c_void_p * count)(*a) if a else None for a in at]
        o = _lib.EgMuon()
        o.rows, o.cols, o.count, o.planes = shape[0], shape[1], count, planes[wt]
        o.params, o.grads, o.momenta = (ctypes.cast(a, ctypes.c_void_p) if a is not None else None for a in arrays)
        o.param_dtype, o.grad_dtype = _DTYPES[wt], _DTYPES[gt]
        o.param_stride[:], o.grad_stride[:] = ws, gs
        if ms is not None:
            o.momentum_stride[:] = ms
        o.coefficients = ctypes.cast(table, ctypes.c_void_p)
        o.steps, o.nesterov = steps, int(nesterov)
        o.momentum, o.eps, o.keep, o.rate = momentum, eps, keep, rate_of(shape)
        need = _lib.load().eg_muon_workspace_size(o.rows, o.cols, count, o.planes)
        if need < 0:
            raise ValueError(f"matrices of {list(shape)}: 1 to 2^20 rows and columns")
        buf = _WS.get(need, dev)
        _lib.call("eg_muon_step", ctypes.byref(o), _lib.ptr(buf), buf.numel(), _lib.stream_ptr(dev))


def muon_step(params, grads, momenta, *, lr: float, weight_decay: float = 0.0, momentum: float = 0.95,
              nesterov: bool = True, steps: int = 5, coefficients=QUINTIC, eps: float = 1e-7,
              products: str | None = None) -> None:
    """One step of ``params`` (a list of f32, bf16 or f16 ``[rows, cols]`` or
    ``[count, rows, cols]``, each matrix an update of its own), in place, with
    ``momenta`` (f32, the same shapes), in place, from ``grads``.  Any strides;
    matrices of one shape, type and strides share their launches.  ``coefficients``:
    one (a, b, c) for every Newton-Schulz step, or one each."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"{len(params)} params, {len(grads)} grads and {len(momenta)} momenta")
    for w, g, m in zip(params, grads, momenta):
        _check(w, "params")
        _check(g, "grads", w)
        _check(m, "momenta", w)
        if m.dtype != torch.float32:
            raise ValueError(f"momenta must be f32, got {m.dtype}")
        _writable(w, "params")
        _writable(m, "momenta")
    table = _coefficients(coefficients, steps)
    planes = {t: _planes(products, t) for t in _DTYPES}
    with torch.no_grad():
        _run(params, grads, momenta, planes, table, steps, momentum=float(momentum), nesterov=nesterov,
             eps=float(eps), keep=1.0 - lr * weight_decay,
             rate_of=lambda shape: lr * max(1.0, shape[0] / shape[1]) ** 0.5)


def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients=QUINTIC, eps: float = 1e-7,
                  out: torch.Tensor | None = None, products: str | None = None) -> torch.Tensor:
    """``x`` (f32, bf16 or f16 ``[rows, cols]`` or ``[count, rows, cols]``) with every matrix's
    singular values driven to about 1, in ``x``'s type.  ``out``: where it is written (``x`` for in place)."""
    _check(x, "x")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _check(out, "out", x)
        _writable(out, "out")
    table = _coefficients(coefficients, steps)
    with torch.no_grad():
        _run([out], [x], None, {out.dtype: _planes(products, out.dtype)}, table, steps, momentum=0.0, nesterov=False,
             eps=float(eps), keep=0.0, rate_of=lambda shape: -1.0)
    return out


class MuonState:
    """Weights and their momenta.  ``params``: ``PleWeights.w_key`` as ``[streams, n, n]``,
    ``w_value``, or other 2-D weights; ``momenta``: f32 tensors to go on from (zeros otherwise)."""

    def __init__(self, params, momenta=None, *, momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
                 coefficients=QUINTIC, eps: float = 1e-7, products: str | None = None):
        self.params = list(params)
        for w in self.params:
            _check(w, "params")
        self.momenta = [torch.zeros(w.shape, dtype=torch.float32, device=w.device) for w in self.params] \
            if momenta is None else list(momenta)
        self._options = dict(momentum=momentum, nesterov=nesterov, steps=steps, coefficients=coefficients, eps=eps,
                             products=products)
        self.step_count = 0

    def step(self, grads, *, lr: float, weight_decay: float = 0.0) -> None:
        """One step of every weight from its gradient."""
        muon_step(self.params, grads, self.momenta, lr=lr, weight_decay=weight_decay, **self._options)
        self.step_count += 1  # only once the step is on its way
