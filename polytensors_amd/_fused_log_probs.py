"""Log probabilities of given tokens, entropies and most probable alternatives of series logits on gfx950.

For logits z(t) over C classes, one streaming pass a row (csrc/token_log_probs_series.inl) gives
``log p = z - logsumexp(z)`` at the row's token, the entropy ``-sum p (*) log p`` and the classes of
the ``top`` largest constant orders with their log-probability series. The log-softmax series is the
reference's (/root/reference/src/polytensors/_plain.py:262-273); it has neither a fused entropy nor
alternatives. Arithmetic is float32 (float64 for float64 logits), as the fused cross entropy's.

Gradients flow from the log probabilities, the entropy and the alternatives' log probabilities to the
logits: ``_SeriesLogProbs`` for PolyTensor logits requiring grad, the operator's coefficient gradients
inside coefficient_autograd.
"""

from typing import NamedTuple, Optional

import torch

from . import _complex, _gate, _ops
from ._fused_cross_entropy import _rows
from ._tensor import PolyTensor

MAX_TOP = 32
_DTYPES = (torch.float16, torch.bfloat16, torch.float32, torch.float64)


class TokenLogProbs(NamedTuple):
    log_probs: PolyTensor
    entropy: PolyTensor
    top_tokens: Optional[torch.Tensor]
    top_log_probs: Optional[PolyTensor]


def why_ineligible(logits, tokens, top, softcap, ignore_index, allow_grad=False):
    if not isinstance(logits, PolyTensor):
        return "logits must be a PolyTensor"
    reason = _gate.common_reason((logits,), allow_plain_grad=allow_grad, complex_ok=True)
    if reason is not None:
        return reason
    if logits.ndim < 1 or logits.shape[-1] == 0:
        return "logits must be (..., C) with at least one class"
    if logits.dtype not in _DTYPES or _gate.real_dtype(logits.coeffs[-1].dtype) != logits.dtype:   # (the higher orders share one)
        return "logits must be float16/bfloat16/float32/float64 in every order"
    if logits.shape[-1] >= 2 ** 31 or logits.numel() // logits.shape[-1] >= 2 ** 31:
        return "more than 2^31 - 1 rows or classes"
    if isinstance(tokens, PolyTensor) or not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64:
        return "tokens must be an ordinary int64 tensor"
    if tokens.shape != logits.shape[:-1] or tokens.device != logits.device:
        return "tokens must have the logits' shape without the classes, on their device"
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        return f"top must be an int in 0..{MAX_TOP} and at most the number of classes"
    if softcap is not None and not (isinstance(softcap, (int, float)) and 0 < softcap < float("inf")):
        return "softcap must be a positive finite number"
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int):
        return "ignore_index must be an int"
    if _complex.has_complex(logits) and (allow_grad or _gate.coefficient_graph(logits)):
        return "gradients along complex directions are not implemented"
    return None


def _series(stacked):
    """The series of a coefficient-stacked result of the operator (disjoint real orders: no checks)."""
    return PolyTensor._wrap(stacked.unbind(0))


class _SeriesLogProbs(torch.autograd.Function):
    """Log probabilities, entropy and (with ``top``) the alternatives' log probabilities of (N, C) logits with
    their gradient series, under wrapper-level autograd."""

    @staticmethod
    def forward(ctx, logits, tokens, ignore_index, softcap, top):
        ctx.set_materialize_grads(False)
        log_probs, entropy, top_tokens, top_log_probs, lse = _ops.token_log_probs_series(
            _rows(logits.coeffs), tokens, ignore_index, softcap, top)
        ctx.save_for_backward(logits, tokens, lse, entropy, top_tokens)
        ctx.meta = (ignore_index, softcap)
        ctx.mark_non_differentiable(top_tokens)
        outputs = (_series(log_probs), _series(entropy.clone()))   # (the entropy is saved: a caller may change its own)
        return (*outputs, top_tokens, _series(top_log_probs)) if top else outputs

    @staticmethod
    def backward(ctx, *gradients):
        if torch.is_grad_enabled():
            raise NotImplementedError("second-order reverse mode through token_log_probs is not implemented")
        logits, tokens, lse, entropy, top_tokens = ctx.saved_tensors
        ignore_index, softcap = ctx.meta
        cots = []
        for g in (gradients[0], gradients[1], gradients[3] if len(gradients) > 2 else None):
            if g is None:
                cots.append([])
                continue
            coeffs = g.coeffs if isinstance(g, PolyTensor) else (g,)
            own = [c.to(lse.dtype).contiguous() for c in coeffs]
            cots.append(own + [torch.zeros_like(own[0]) for _ in range(logits.degree + 1 - len(own))])
        if not any(cots):
            return None, None, None, None, None
        dz = _ops.token_log_probs_series_backward(_rows(logits.coeffs), tokens, ignore_index, softcap, lse, entropy,
                                                  top_tokens, *cots)
        return _series(dz), None, None, None, None


def _run(logits, tokens, ignore_index, softcap, top):
    """(log_probs, entropy[, top_tokens, top_log_probs]) of (N, C) real-direction logits."""
    if _gate.wrapper_grad(logits):
        return _SeriesLogProbs.apply(logits, tokens, ignore_index, softcap, top)
    log_probs, entropy, top_tokens, top_log_probs, _ = _ops.token_log_probs_series(_rows(logits.coeffs), tokens, ignore_index,
                                                                                   softcap, top)
    outputs = (_series(log_probs), _series(entropy))
    return (*outputs, top_tokens, _series(top_log_probs)) if top else outputs


def _complex_run(logits, tokens, ignore_index, softcap, top):
    """The same along complex directions: the real runs' results side by side, combined."""
    ids = []

    def side_by_side(z):
        y = _run(z, tokens, ignore_index, softcap, top)
        ids.append(y[2] if top else None)   # (the constant order is every run's)
        parts = [y[0], y[1]] + ([y[3]] if top else [])
        return PolyTensor(tuple(torch.cat([p.coeffs[k].reshape(tokens.shape[0], -1) for p in parts], 1)
                                for k in range(z.degree + 1)))

    y = _complex.at_real_nodes(side_by_side, "token_log_probs", logits)
    outputs = (y[:, 0], y[:, 1])
    return (*outputs, ids[0], y[:, 2:]) if top else outputs


def token_log_probs(logits, tokens, top=0, softcap=None, ignore_index=-100):
    """``PolyTensor.token_log_probs``."""
    reason = why_ineligible(logits, tokens, top, softcap, ignore_index, allow_grad=_gate.wrapper_grad(logits))
    if reason is not None:
        raise NotImplementedError(f"token_log_probs: {reason}")
    flat = logits if logits.ndim == 2 else logits.reshape(-1, logits.shape[-1])
    run = _complex_run if _complex.has_complex(logits) else _run
    outputs = run(flat, tokens.reshape(-1).contiguous(), ignore_index, float(softcap or 0.0), top)
    if logits.ndim != 2:
        lead = tuple(tokens.shape)
        outputs = tuple(y.reshape(lead if i < 2 else (*lead, top)) for i, y in enumerate(outputs))
    return TokenLogProbs(*outputs) if top else TokenLogProbs(*outputs, None, None)
