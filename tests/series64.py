"""Plain float64 series arithmetic and the operators' definitions in it (test helper).

A series is a list of tensors, one per order; every function is made of torch operations that autograd
follows, so coefficient gradients come from reverse mode over the definitions.
"""

import numpy as np
import torch


def mul(a, b):
    return [sum(a[i] * b[k - i] for i in range(k + 1)) for k in range(len(a))]


def log(s):
    out = [s[0].log()]
    for k in range(1, len(s)):
        out.append((k * s[k] - sum(i * out[i] * s[k - i] for i in range(1, k))) / (k * s[0]))
    return out


def exp(u):
    out = [u[0].exp()]
    for k in range(1, len(u)):
        out.append(sum(j * u[j] * out[k - j] for j in range(1, k + 1)) / k)
    return out


def power(s, p):
    """s^p: k s_0 y_k = sum_j ((p + 1) j - k) s_j y_{k-j}."""
    y = [s[0] ** p]
    for k in range(1, len(s)):
        y.append(sum(((p + 1) * j - k) * s[j] * y[k - j] for j in range(1, k + 1)) / (k * s[0]))
    return y


def tanh(u):
    e = exp([2 * c for c in u])
    inverse = power([e[0] + 1] + e[1:], -1.0)
    return [1 - 2 * inverse[0]] + [-2 * c for c in inverse[1:]]


def rotate(x, cos, sin, interleaved):
    """x (..., L, H, D) with cos, sin (..., L, R / 2)."""
    half = cos.shape[-1]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def norm_rope(x, w, cos, sin, positions, eps, interleaved):
    """Series x (B, L, H, D), weight series w or None, positions (B, L): the series (B, H, L, D)."""
    square = [c.mean(-1, keepdim=True) for c in mul(x, x)]
    square[0] = square[0] + eps
    n = mul(x, power(square, -0.5))
    if w is not None:
        n = mul(n, w) if len(w) == len(x) else [c * w[0] for c in n]
    c, s = cos[positions.clamp_min(0)], sin[positions.clamp_min(0)]
    keep = (positions >= 0)[..., None, None]
    return [torch.where(keep, rotate(v, c, s, interleaved), 0.0).transpose(-2, -3) for v in n]


def log_probs(z, tokens, top=0, softcap=None, ignore_index=-100):
    """Series z (N, C): log probabilities and entropies (N,), alternatives (N, top) and their log probabilities."""
    masked = (z[0] == -float("inf")) & (softcap is None)
    raw = z[0]
    u = [torch.where(masked, 0.0 if k else -1e300, c) for k, c in enumerate(z)]
    if softcap is not None:
        u = [softcap * c for c in tanh([c / softcap for c in z])]
    m = u[0].detach().amax(1, keepdim=True)
    e = exp([u[0] - m] + u[1:])
    lse = log([c.sum(1, keepdim=True) for c in e])
    lse[0] = lse[0] + m
    logp = [a - b for a, b in zip(u, lse)]
    entropy = [-c.sum(1) for c in mul(exp(logp), logp)]
    if softcap is None:   # a masked class as it is asked for: -inf, and the logits' own higher orders
        logp = [a - b for a, b in zip(z, lse)]
    ignored = tokens == ignore_index
    at = tokens.masked_fill(ignored, 0)[:, None]
    out = [[torch.where(ignored, 0.0, c.gather(1, at)[:, 0]) for c in logp], [torch.where(ignored, 0.0, c) for c in entropy]]
    if top:
        ids = torch.sort(raw.detach(), dim=1, descending=True, stable=True).indices[:, :top]
        out += [torch.where(ignored[:, None], -1, ids), [torch.where(ignored[:, None], 0.0, c.gather(1, ids)) for c in logp]]
    return out


def philox(first, count, seed):
    """Words of Philox4x32-10 for elements first .. first + count - 1: word i mod 4 of block i // 4."""
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.arange(first // 4, (first + count + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> shift, np.zeros_like(block), np.zeros_like(block)]
    seed %= 2 ** 64
    for i in range(10):
        k0 = np.uint64((seed % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32)
        k1 = np.uint64((seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ k0, b & low, (a >> shift) ^ c[3] ^ k1, a & low]
    return np.stack(c, 1).reshape(-1)[first % 4:first % 4 + count]


def keep(first, count, seed, p):
    return torch.from_numpy(philox(first, count, seed) >= np.uint64(int(p * 2.0 ** 32)))
