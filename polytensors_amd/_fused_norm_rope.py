"""RMSNorm of every head of queries and keys, and their rotation by position, on gfx950.

For heads x(t) at position pos:  y(t) = R(pos) (w(t) * x(t) * rsqrt(mean(x(t)^2) + eps)), read from
the projection's (B, L, H, D) and written as the attention's (B, H, L, D), both operands in one launch
(csrc/norm_rope_series.inl). The reference has no such operation: there it is F.rms_norm
(/root/reference/src/polytensors/_decompositions.py:14-22), slices, products with the tables and a
transposing copy, each a pass over every order.

Gradients: a PolyTensor operand or weight requiring grad records ``_SeriesNormRope``; inside
coefficient_autograd the operator records coefficient gradients, an ordinary weight's among them.
"""

import torch

from . import _complex, _gate, _ops
from ._tensor import PolyTensor

MAX_HEAD = 256
_DTYPES = (torch.float16, torch.bfloat16, torch.float32, torch.float64)


def why_ineligible(query, key, cos, sin, positions, query_weight, key_weight, eps):
    operands = [x for x in (query, key, query_weight, key_weight) if x is not None]
    if query is None or key is None or not all(isinstance(x, torch.Tensor) for x in (*operands, cos, sin)):
        return "query, key, cos, sin and the weights must be tensors"
    reason = _gate.common_reason(operands, allow_plain_grad=_gate.wrapper_grad(*operands), complex_ok=True)
    if reason is not None:
        return reason
    dtype, device = query.dtype, query.device   # (a series' dtype is its constant order's, real here)
    if dtype not in _DTYPES:
        return f"dtype {dtype} is not supported (float32, float64, bfloat16 or float16)"
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    grads = torch.is_grad_enabled()
    for x in operands:   # (a series' higher orders share one dtype: its last order stands for them)
        series = isinstance(x, PolyTensor)
        if x.dtype != dtype or (series and x.coeffs[-1].dtype != dtype and _gate.real_dtype(x.coeffs[-1].dtype) != dtype):
            return "query, key and the weights must share one dtype"
        if x.device != device:
            return "operands and weights must be on one device"
        if not series:
            if grads and _gate.wrapper_grad(x):
                return ("an ordinary (non-PolyTensor) operand or weight requires grad: its gradient would be a series, which "
                        "autograd cannot hand to it (make it a PolyTensor, or use coefficient_autograd)")
            if _gate.transformed(x):
                return "function transforms are not supported"
    shape, key_shape = query.shape, key.shape
    if len(shape) != 4 or len(key_shape) != 4 or shape[:2] != key_shape[:2] or shape[3] != key_shape[3]:
        return "query and key must be (B, L, H, D) and (B, L, G, D)"
    batch, length, heads, dim = shape
    if not 1 <= dim <= MAX_HEAD or heads == 0 or key_shape[2] == 0:
        return f"heads of 1..{MAX_HEAD} elements, at least one head each"
    if max(heads, key_shape[2]) * batch * length >= 2 ** 31:
        return "more than 2^31 - 1 heads"
    for w in (query_weight, key_weight):
        if w is not None and tuple(w.shape) != (dim,):
            return "weights must be (D,)"
    for t in (cos, sin):
        if isinstance(t, PolyTensor) or t.dtype != acc or t.device != device or t.ndim != 2 or t.shape != cos.shape \
                or 2 * t.shape[1] > dim:
            return f"cos and sin must be ordinary {acc} (P, rotary / 2) on the operands' device, rotary at most D"
        if _gate.transformed(t):
            return "function transforms are not supported"
        if grads and t.requires_grad:
            return "no gradient flows to the cos and sin tables"
    if positions is not None and (
            isinstance(positions, PolyTensor) or not isinstance(positions, torch.Tensor) or positions.dtype != torch.int64 or
            positions.device != device or tuple(positions.shape) not in ((length,), (1, length), (batch, length))):
        return "positions must be an ordinary int64 (L,) or (B, L) on the operands' device"
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0.0 <= eps < float("inf"):
        return "eps must be a finite number of at least 0"
    return None


def _heads(coeffs):
    """Coefficients with one common set of strides and a head's elements side by side (else copies)."""
    strides = coeffs[0].stride()
    if (strides[-1] == 1 or coeffs[0].shape[-1] <= 1) and all(c.stride() == strides for c in coeffs[1:]):
        return list(coeffs)
    return [c.contiguous() for c in coeffs]


def _weight(w):
    return [] if w is None else [c.contiguous() for c in _gate.coefficients(w, 0)]


class _SeriesNormRope(torch.autograd.Function):
    """The operation with its gradient series, under wrapper-level autograd. ``key`` may be None."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, cos, sin, positions, eps, interleaved):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(query, key, query_weight, key_weight, cos, sin, positions)
        ctx.meta = (eps, interleaved)
        q, k = _ops.norm_rope_series(_heads(query.coeffs), [] if key is None else _heads(key.coeffs), cos, sin, positions,
                                     _weight(query_weight), _weight(key_weight), eps, interleaved)
        if key is None:
            return PolyTensor.from_stacked(q)
        return PolyTensor.from_stacked(q), PolyTensor.from_stacked(k)

    @staticmethod
    def backward(ctx, *gradients):
        if torch.is_grad_enabled():
            raise NotImplementedError("second-order reverse mode through qk_norm_rope is not implemented")
        query, key, query_weight, key_weight, cos, sin, positions = ctx.saved_tensors
        eps, interleaved = ctx.meta
        operands = []
        for x, w, g, need in ((query, query_weight, gradients[0], ctx.needs_input_grad[2]),
                              (key, key_weight, gradients[-1], ctx.needs_input_grad[3])):
            if x is None or g is None:
                operands.append(([], None, [], False))
                continue
            cots = list(g.coeffs) if isinstance(g, PolyTensor) else [g]
            cots = [c.to(x.dtype) for c in cots] + [None] * (x.degree + 1 - len(cots))
            operands.append((_heads(x.coeffs), cots, _weight(w), need))
        results = _ops.norm_rope_gradients(operands, cos, sin, positions, eps, interleaved)
        dx = [None if r is None else PolyTensor.from_stacked(r[0]) for r in results]
        dw = [None if r is None or r[1] is None else PolyTensor.from_stacked(r[1]) for r in results]
        return (*dx, *dw, None, None, None, None, None)


def _run(query, key, query_weight, key_weight, cos, sin, positions, eps, interleaved):
    """The operation on real series or ordinary tensors of one kind (key None: queries alone)."""
    recorded = False
    if torch.is_grad_enabled():
        if _gate.wrapper_grad(query, key, query_weight, key_weight):
            return _SeriesNormRope.apply(query, key, query_weight, key_weight, cos, sin, positions, eps, interleaved)
        recorded = _gate.coefficient_graph(query, key, query_weight, key_weight)
    series = isinstance(query, PolyTensor)
    q, k = _heads(_gate.coefficients(query, 0)), [] if key is None else _heads(_gate.coefficients(key, 0))
    args = (q, k, cos, sin, positions, _weight(query_weight), _weight(key_weight), eps, interleaved)
    if recorded:
        out = _ops.norm_rope_series_orders(*args)
        parts = [out[:len(q)], out[len(q):]]
    else:
        parts = [y.unbind(0) for y in _ops.norm_rope_series(*args)]
    results = [PolyTensor._wrap(tuple(p)) if series else p[0] for p in parts[:1 if key is None else 2]]
    return results[0] if key is None else tuple(results)


def _single(x, w, cos, sin, positions, eps, interleaved):
    return _run(x, None, w, None, cos, sin, positions, eps, interleaved)


def qk_norm_rope(query, key, cos, sin, positions=None, query_weight=None, key_weight=None, eps=None, interleaved=False):
    """``PolyTensor.qk_norm_rope``."""
    if eps is None and isinstance(query, torch.Tensor) and _gate.real_dtype(query.dtype).is_floating_point:
        eps = torch.finfo(_gate.real_dtype(query.dtype)).eps
    reason = why_ineligible(query, key, cos, sin, positions, query_weight, key_weight, eps)
    if reason is not None:
        raise NotImplementedError(f"qk_norm_rope: {reason}")
    cos, sin, eps, interleaved = cos.contiguous(), sin.contiguous(), float(eps), bool(interleaved)
    if positions is not None:
        positions = (positions.reshape(-1) if positions.ndim == 2 and positions.shape[0] == 1 else positions).contiguous()
    degree = next(x.degree for x in (query, key, query_weight, key_weight) if isinstance(x, PolyTensor))
    if not isinstance(query, PolyTensor) and isinstance(query_weight, PolyTensor):
        query = PolyTensor.constant(query, degree)
    if not isinstance(key, PolyTensor) and isinstance(key_weight, PolyTensor):
        key = PolyTensor.constant(key, degree)
    complex_directions = _complex.has_complex(query, key, query_weight, key_weight)
    if isinstance(query, PolyTensor) and isinstance(key, PolyTensor) and not complex_directions:
        return _run(query, key, query_weight, key_weight, cos, sin, positions, eps, interleaved)
    outputs = []   # an ordinary operand beside a series, or complex directions: an operand at a time
    for x, w in ((query, query_weight), (key, key_weight)):
        if _complex.has_complex(x, w):
            outputs.append(_complex.at_real_nodes(_single, "qk_norm_rope", x, w, cos, sin, positions, eps, interleaved))
        else:
            outputs.append(_single(x, w, cos, sin, positions, eps, interleaved))
    return tuple(outputs)
