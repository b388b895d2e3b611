"""Dropout of a degree-K series on gfx950: one mask for every order, from a counter-based generator.

``y_k = x_k m / (1 - p)`` with m a function of a seed and the element's index (Philox4x32-10,
csrc/dropout_series.inl), so that the gradient draws the mask again instead of reading a stored one.
The reference's rule stores the mask of the constant order and multiplies each order by it
(/root/reference/src/polytensors/_dispatch.py); here the orders pass once through one kernel.
The operation is linear in the series and acts on each order alone: complex orders are two real
buffers under the same mask, and its gradient differentiates again.
"""

import math

import torch

from . import _gate, _ops
from ._tensor import PolyTensor

_DTYPES = (torch.float16, torch.bfloat16, torch.float32, torch.float64)
_MAX_BUFFERS = _gate.MAX_ELEMENTWISE_DEGREE + 1   # a call of the operator


def why_ineligible(input, p, seed, allow_grad=False):
    if not isinstance(input, PolyTensor):
        return "the input must be a PolyTensor"
    reason = _gate.common_reason((input,), allow_plain_grad=allow_grad, complex_ok=True, complex_base_ok=True,
                                 max_degree=_gate.MAX_ELEMENTWISE_DEGREE)
    if reason is not None:
        return reason
    if any(_gate.real_dtype(c.dtype) not in _DTYPES or _gate.real_dtype(c.dtype) != _gate.real_dtype(input.dtype)
           for c in input.coeffs):
        return "coefficients must be float16/bfloat16/float32/float64 (or their complex types) of one precision"
    if isinstance(seed, torch.Tensor) and (isinstance(seed, PolyTensor) or seed.dtype != torch.int64 or
                                           seed.numel() != 1 or seed.device != input.device):
        return "the seed must be an int or one int64 on the input's device"
    return None


def _apply(coeffs, seed, p, recorded=False):
    """Every coefficient's dropout; ``recorded``: as a tensor per order, which autograd records."""
    planes = []   # real buffers, two for a complex order
    for c in coeffs:
        planes += [c.real.contiguous(), c.imag.contiguous()] if c.is_complex() else [c.contiguous()]
    out = []
    for i in range(0, len(planes), _MAX_BUFFERS):
        part = planes[i:i + _MAX_BUFFERS]
        out += _ops.dropout_series_orders(part, seed, p) if recorded else _ops.dropout_series(part, seed, p).unbind(0)
    out = iter(out)
    return tuple(torch.complex(next(out), next(out)) if c.is_complex() else next(out) for c in coeffs)


class _SeriesDropout(torch.autograd.Function):
    """Dropout under wrapper-level autograd: the same mask on the cotangent series."""

    @staticmethod
    def forward(ctx, input, seed, p):
        ctx.save_for_backward(seed)
        ctx.p = p
        return PolyTensor._wrap(_apply(input.coeffs, seed, p))

    @staticmethod
    def backward(ctx, gradient):
        (seed,) = ctx.saved_tensors
        if torch.is_grad_enabled() and gradient.requires_grad:
            return _SeriesDropout.apply(gradient, seed, ctx.p), None, None
        if not isinstance(gradient, PolyTensor):
            return _apply((gradient,), seed, ctx.p)[0], None, None
        return PolyTensor._wrap(_apply(gradient.coeffs, seed, ctx.p)), None, None


def dropout(input, p=0.5, seed=None):
    """``PolyTensor.dropout``."""
    if isinstance(p, bool) or not isinstance(p, (int, float)) or not (math.isfinite(p) and 0.0 <= p <= 1.0):
        raise ValueError(f"dropout: p must be in [0, 1], got {p!r}")
    if seed is not None and not isinstance(seed, torch.Tensor):
        if isinstance(seed, bool) or not isinstance(seed, int) or not -2 ** 63 <= seed < 2 ** 63:
            raise ValueError("dropout: the seed must be a 64-bit int or an int64 tensor of one element")
    grads = _gate.wrapper_grad(input)
    reason = why_ineligible(input, p, seed, allow_grad=grads)
    if reason is not None:
        raise NotImplementedError(f"dropout: {reason}")
    if seed is None:
        seed = torch.empty(1, dtype=torch.int64, device=input.device).random_()
    elif not isinstance(seed, torch.Tensor):
        seed = torch.full((1,), seed, dtype=torch.int64, device=input.device)
    if grads:
        return _SeriesDropout.apply(input, seed, float(p))
    return PolyTensor._wrap(_apply(input.coeffs, seed, float(p), recorded=_gate.coefficient_graph(input)))


def functional(input, p, training, inplace):
    """``torch.nn.functional.dropout`` on a PolyTensor: the input itself outside training or at p = 0."""
    if p < 0.0 or p > 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
    if not training or p == 0:
        return input
    if inplace:
        raise NotImplementedError("dropout: inplace=True is not supported on a PolyTensor")
    return dropout(input, float(p))
