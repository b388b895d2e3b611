"""A decoder's step with the operators together: projection, norm and rotation of queries and keys, attention,
dropout, output projection, token log probabilities and entropy; values and gradients in float64 against the
definitions in plain series arithmetic.

Tolerance 1e-10 of an order's largest value: about 10^5 roundings of 2^-53 and an order of magnitude for
the condition of two products and a softmax between them.
"""

import math

import pytest
import torch
import torch.nn.functional as F

from polytensors_amd import PolyTensor
from tests import series64

pytestmark = pytest.mark.gpu

B, L, H, D, C, DEGREE, P, SEED = 2, 9, 2, 16, 50, 2, 0.25, 77


def _inputs(dtype=torch.float64):
    g = torch.Generator().manual_seed(1)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g, dtype=torch.float64) * scale).to(dtype)   # noqa: E731
    E = H * D
    x = [n(B, L, E, scale=0.5 ** k) for k in range(DEGREE + 1)]
    weights = [n(3 * E, E, scale=E ** -0.5), n(D, scale=0.1) + 1, n(D, scale=0.1) + 1, n(C, E, scale=E ** -0.5)]
    angle = torch.arange(L, dtype=torch.float64)[:, None] * 10.0 ** (-torch.arange(0, D, 2).double() / D)
    tokens = torch.randint(0, C, (B, L), generator=g)
    tokens[0, -2:] = -100
    return x, weights, angle.cos().to(dtype), angle.sin().to(dtype), tokens


def _block(x, wqkv, wq, wk, wout, cos, sin, tokens):
    """The step as a program writes it; returns TokenLogProbs."""
    qkv = F.linear(x, wqkv).reshape(B, L, 3 * H, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]
    q, k = PolyTensor.qk_norm_rope(q, k, cos, sin, query_weight=wq, key_weight=wk, eps=1e-6)
    y = F.scaled_dot_product_attention(q, k, v.transpose(1, 2), is_causal=True)
    y = PolyTensor.dropout(y.transpose(1, 2).reshape(B, L, H * D), P, seed=SEED)
    return PolyTensor.token_log_probs(F.linear(x + y, wout), tokens, top=3)


def _reference(x, wqkv, wq, wk, wout, cos, sin, tokens):
    qkv = [(c @ wqkv.t()).view(B, L, 3 * H, D) for c in x]
    positions = torch.arange(L).expand(B, L)
    q = series64.norm_rope([c[:, :, :H] for c in qkv], [wq], cos, sin, positions, 1e-6, False)
    k = series64.norm_rope([c[:, :, H:2 * H] for c in qkv], [wk], cos, sin, positions, 1e-6, False)
    v = [c[:, :, 2 * H:].transpose(1, 2) for c in qkv]
    n = DEGREE + 1
    scores = [sum(q[i] @ k[o - i].transpose(-1, -2) for i in range(o + 1)) / math.sqrt(D) for o in range(n)]
    later = torch.ones(L, L).triu(1).bool()
    e = series64.exp(scores)
    e = [c.masked_fill(later, 0.0) for c in e]
    inverse = series64.power([c.sum(-1, keepdim=True) for c in e], -1.0)
    p = series64.mul(e, inverse)
    y = [sum(p[i] @ v[o - i] for i in range(o + 1)).transpose(1, 2).reshape(B, L, H * D) for o in range(n)]
    kept = series64.keep(0, y[0].numel(), SEED, P).view(y[0].shape)
    y = [torch.where(kept, c / (1 - P), 0.0) for c in y]
    logits = [((a + b) @ wout.t()).flatten(0, 1) for a, b in zip(x, y)]
    return series64.log_probs(logits, tokens.flatten(), top=3)


def _close(got, want, what):
    got, want = got.detach().cpu().double(), want.detach()
    assert (got.reshape(want.shape) - want).abs().max() <= 1e-10 * max(1.0, want.abs().max().item()), what


def _objective(log_probs, entropy):
    return [a.sum() + 0.1 * b.sum() for a, b in zip(log_probs, entropy)]


def test_step_and_its_coefficient_gradients():
    x, weights, cos, sin, tokens = _inputs()
    x64 = [c.clone().requires_grad_() for c in x]
    w64 = [w.clone().requires_grad_() for w in weights]
    want = _reference(x64, *w64, cos, sin, tokens)
    leaves, params = [c.cuda().requires_grad_() for c in x], [w.cuda().requires_grad_() for w in weights]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        got = _block(PolyTensor(tuple(leaves)), *params, cos.cuda(), sin.cuda(), tokens.cuda())
        mine = _objective(got.log_probs.coeffs, got.entropy.coeffs)
    assert torch.equal(got.top_tokens.cpu().flatten(0, 1), want[2])
    for k in range(DEGREE + 1):
        _close(got.log_probs.coeffs[k], want[0][k], "log_probs")
        _close(got.entropy.coeffs[k], want[1][k], "entropy")
        _close(got.top_log_probs.coeffs[k], want[3][k], "top_log_probs")
    weights_of_orders = [1.0, 0.5, -0.25]
    total = sum(w * c for w, c in zip(weights_of_orders, mine))
    grads = torch.autograd.grad(total, leaves + params)
    ref = torch.autograd.grad(sum(w * c for w, c in zip(weights_of_orders, _objective(want[0], want[1]))), x64 + w64)
    for i, (a, b) in enumerate(zip(grads, ref)):
        _close(a, b, f"gradient {i}")


def test_step_in_wrapper_reverse_mode():
    x, weights, cos, sin, tokens = _inputs()
    x64 = [c.clone().requires_grad_() for c in x]
    want = _reference(x64, *weights, cos, sin, tokens)
    X = PolyTensor(tuple(c.cuda() for c in x), requires_grad=True)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        got = _block(X, *(w.cuda() for w in weights), cos.cuda(), sin.cuda(), tokens.cuda())
        (got.log_probs.sum() + got.entropy.sum() * 0.1).backward()
        # the gradient series of the objective: coefficient i is d(objective_K) / d x_{K - i}
        objective = _objective(want[0], want[1])
        ref = torch.autograd.grad(objective[DEGREE], x64)
        for i in range(DEGREE + 1):
            _close(X.grad.coeffs[i], ref[DEGREE - i], f"order {i}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_in_the_other_types_runs_and_has_gradients(dtype):
    x, weights, cos, sin, tokens = _inputs(dtype)
    X = PolyTensor(tuple(c.cuda() for c in x), requires_grad=True)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        got = _block(X, *(w.cuda() for w in weights), cos.float().cuda(), sin.float().cuda(), tokens.cuda())
        (got.log_probs.mean() - got.entropy.mean()).backward()
        assert all(c.isfinite().all() and c.abs().sum() > 0 for c in X.grad.coeffs)
