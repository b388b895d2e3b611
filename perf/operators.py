"""What a decoder's training and serving steps call around its attention and its loss, as cases that are
timed and checked: the per-head RMSNorm of queries and keys with the position rotation, dropout from a
counter-based generator, and the log probabilities of given tokens with the entropy and the most probable
alternatives, each on degree-K Taylor series (one tensor per order), forward and with gradients.

With ``own`` false ``run`` computes them in elementary torch operations (float32, or float64 for float64
inputs, rounded once at the end); with ``own`` true it calls this package's operators. ``exact`` restates
the definitions in 64 bits: the series by other recurrences than the plain form's, the gradients by
torch's own reverse mode over them, the random numbers in numpy.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # a step of generation: one new token of each of 32 sequences, all at positions of their own, heads shared
        # by groups of queries; a launch or two is what it should take
        dict(name="qk_step_bf16", kind="qk", dtype="bf16", degree=2, batch=32, length=1, heads=32, kv_heads=8, head=128,
             rotary=128, interleaved=False, table=8192, grad=False),
        # prefill at the sizes of the attention benchmark: 4 sequences of 2048, 16 heads of 128, degree 4
        dict(name="qk_prefill_bf16", kind="qk", dtype="bf16", degree=4, batch=4, length=2048, heads=16, kv_heads=16,
             head=128, rotary=128, interleaved=False, table=2048, grad=False),
        # a training step: the gradients of every coefficient of both operands and of both weights
        dict(name="qk_train_bf16", kind="qk", dtype="bf16", degree=3, batch=2, length=2048, heads=32, kv_heads=8, head=128,
             rotary=128, interleaved=False, table=2048, grad=True),
        # a head that is no power of two, a quarter of it rotated in neighbouring pairs, an odd length
        dict(name="qk_partial_f32", kind="qk", dtype="f32", degree=3, batch=3, length=1001, heads=12, kv_heads=12, head=80,
             rotary=20, interleaved=True, table=2048, grad=True),
        # serving: the sampled tokens of 8 sequences over a large vocabulary, with 20 alternatives; few long rows
        dict(name="logprob_step_bf16", kind="logprob", dtype="bf16", degree=1, rows=8, classes=131072, top=20, softcap=None,
             grad=False),
        # scoring a batch at the size of the cross-entropy benchmark, five alternatives a token
        dict(name="logprob_score_f32", kind="logprob", dtype="f32", degree=4, rows=8192, classes=32000, top=5, softcap=None,
             grad=False),
        # a training step on log probabilities with an entropy term (a policy's), a vocabulary of no whole vectors
        dict(name="logprob_train_bf16", kind="logprob", dtype="bf16", degree=3, rows=4096, classes=32001, top=0, softcap=None,
             grad=True),
        # a short batch with capped logits in float16, gradients through the alternatives too (distillation)
        dict(name="logprob_capped_f16", kind="logprob", dtype="f16", degree=2, rows=257, classes=50257, top=8, softcap=30.0,
             grad=True),
        # the smallest: one short sequence's activations
        dict(name="dropout_small_bf16", kind="dropout", dtype="bf16", degree=2, rows=16, width=768, p=0.1, grad=False),
        # the residual branch of the benchmark decoder (8 x 1024 tokens, width 768) in a training step
        dict(name="dropout_decoder_f32", kind="dropout", dtype="f32", degree=3, rows=8192, width=768, p=0.1, grad=True),
        # the activations of the norm benchmark
        dict(name="dropout_wide_bf16", kind="dropout", dtype="bf16", degree=4, rows=8192, width=4096, p=0.2, grad=True),
        # rows of odd length in float64
        dict(name="dropout_odd_f64", kind="dropout", dtype="f64", degree=1, rows=1001, width=1023, p=0.5, grad=False),
    ]


def _log(rng, low, high, multiple=1):
    """A size between low and high, even over its logarithm; odd ones among them."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(1, int(round(v / multiple))) * multiple


def _drawn(rng):
    dtype = rng.choice(["f32", "f32", "bf16", "bf16", "bf16", "f16", "f64"])
    degree = rng.choice([1, 1, 2, 2, 3, 3, 4, 5])
    kind = rng.choice(["qk", "logprob", "dropout"])
    c = dict(kind=kind, dtype=dtype, degree=degree)
    if kind == "qk":
        head = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, rng.randrange(16, 200)])
        rotary = rng.choice([head // 2 * 2, head // 2 * 2, head // 4 * 2, head // 8 * 2 or 2])
        kv = rng.choice([1, 2, 4, 8])
        length = 1 if rng.random() < 0.3 else _log(rng, 2, 4096)
        batch = _log(rng, 1, 256) if length == 1 else rng.choice([1, 2, 3, 4, 8])
        return dict(c, batch=batch, length=length, heads=kv * rng.choice([1, 1, 2, 4]), kv_heads=kv, head=head, rotary=rotary,
                    interleaved=rng.random() < 0.4, table=_log(rng, max(length, 64), 16384), grad=length > 1 and rng.random() < 0.5)
    if kind == "logprob":
        rows = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 8192)
        return dict(c, rows=rows, classes=_log(rng, 256, 262144, rng.choice([1, 1, 8, 64])), top=rng.choice([0, 1, 5, 20, 32]),
                    softcap=rng.choice([None, None, 30.0]), grad=rng.random() < 0.5)
    return dict(c, rows=_log(rng, 1, 16384), width=_log(rng, 64, 8192, rng.choice([1, 8, 64])),
                p=rng.choice([0.05, 0.1, 0.3, 0.5]), grad=rng.random() < 0.5)


def _cost(case):
    # (the plain form and the 64-bit results hold several temporaries of the inputs' size)
    return work(case)["bytes"] / SIZES[case["dtype"]]


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        c = _drawn(rng)
        if _cost(c) <= 0.5 * top:
            return c


# ---------------------------------------------------------------------------
# Inputs: normal values, coefficient k scaled by 0.5^k; tables, weights and seeds as a program keeps them

EPS = 1e-6


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, K = DTYPES[case["dtype"]], case["degree"]
    acc = torch.float64 if dtype == torch.float64 else torch.float32

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(to)

    def series(*shape, scale=1.0, to=dtype):
        return [normal(*shape, scale=scale * 0.5 ** k, to=to) for k in range(K + 1)]

    if case["kind"] == "qk":
        B, L, H, G, D, R, P = (case[k] for k in ("batch", "length", "heads", "kv_heads", "head", "rotary", "table"))
        # a projection's output holds queries, keys and values side by side; the operator reads its parts in place
        rows = [r.view(B, L, H + 2 * G, D) for r in series(B, L, (H + 2 * G) * D)]
        t = dict(q=[r[:, :, :H] for r in rows], k=[r[:, :, H:H + G] for r in rows],
                 wq=1 + normal(D, scale=0.1), wk=1 + normal(D, scale=0.1))
        angle = torch.arange(P, device=DEV, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
        t["cos"], t["sin"] = angle.cos().to(acc), angle.sin().to(acc)
        if L == 1:   # a step: every sequence at a position of its own
            t["positions"] = torch.randint(0, P, (B, 1), generator=g, device=DEV)
        else:        # a batch of sequences that start anywhere in the table
            start = torch.randint(0, P - L + 1, (B, 1), generator=g, device=DEV)
            t["positions"] = start + torch.arange(L, device=DEV)
        if case["grad"]:
            t["cq"], t["ck"] = series(B, H, L, D), series(B, G, L, D)
        return t
    if case["kind"] == "logprob":
        N, C, top = case["rows"], case["classes"], case["top"]
        t = dict(z=series(N, C, scale=2.0), tokens=torch.randint(0, C, (N,), generator=g, device=DEV))
        if N > 4:    # a padded batch: some rows have no token
            t["tokens"][torch.randint(0, N, (N // 16 + 1,), generator=g, device=DEV)] = -100
        if case["grad"]:
            t["cl"], t["ch"] = series(N, to=acc), series(N, scale=0.1, to=acc)
            if top:
                t["ct"] = series(N, top, scale=0.5, to=acc)
        return t
    t = dict(x=series(case["rows"], case["width"]),
             seed=torch.randint(-2 ** 62, 2 ** 62, (1,), generator=g, device=DEV))
    if case["grad"]:
        t["c"] = series(case["rows"], case["width"])
    return t


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    from polytensors_amd import PolyTensor

    if case["kind"] == "qk":
        if case["grad"]:   # coefficients and weights are ordinary autograd leaves
            for n in ("q", "k"):
                s[n] = [c.detach().requires_grad_() for c in s[n]]
            for n in ("wq", "wk"):
                s[n] = s[n].requires_grad_()
        s["Q"], s["K"] = PolyTensor(tuple(s["q"])), PolyTensor(tuple(s["k"]))
    elif case["kind"] == "logprob":
        s["Z"] = PolyTensor(tuple(s["z"]), requires_grad=case["grad"])
        if case["grad"]:
            s["C"] = [PolyTensor(tuple(s[n])) for n in ("cl", "ch", "ct") if n in s]
    else:
        s["X"] = PolyTensor(tuple(s["x"]), requires_grad=case["grad"])
        if case["grad"]:
            s["C"] = PolyTensor(tuple(s["c"]))
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"qk": _own_qk, "logprob": _own_logprob, "dropout": _own_dropout}[kind](state)
    return {"qk": _plain_qk, "logprob": _plain_logprob, "dropout": _plain_dropout}[kind](state)


# ---------------------------------------------------------------------------
# The package's operators, as a program calls them

def _own_qk(s):
    from polytensors_amd import PolyTensor

    args = (s["Q"], s["K"], s["cos"], s["sin"])
    kw = dict(positions=s["positions"], query_weight=s["wq"], key_weight=s["wk"], eps=EPS,
              interleaved=s["case"]["interleaved"])
    if not s["case"]["grad"]:
        with torch.no_grad(), PolyTensor.plain_range():
            q, k = PolyTensor.qk_norm_rope(*args, **kw)
        return dict(q=list(q.coeffs), k=list(k.coeffs))
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        q, k = PolyTensor.qk_norm_rope(*args, **kw)
    n = len(s["q"])
    grads = torch.autograd.grad((*q.coeffs, *k.coeffs), (*s["q"], *s["k"], s["wq"], s["wk"]), (*s["cq"], *s["ck"]))
    return dict(q=[c.detach() for c in q.coeffs], k=[c.detach() for c in k.coeffs], dq=list(grads[:n]),
                dk=list(grads[n:2 * n]), dwq=grads[-2], dwk=grads[-1])


def _own_logprob(s):
    from polytensors_amd import PolyTensor

    case = s["case"]
    if not case["grad"]:
        with torch.no_grad(), PolyTensor.plain_range():
            y = PolyTensor.token_log_probs(s["Z"], s["tokens"], top=case["top"], softcap=case["softcap"])
        out, grads = y, None
    else:
        with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
            y = PolyTensor.token_log_probs(s["Z"], s["tokens"], top=case["top"], softcap=case["softcap"])
            parts = [y.log_probs, y.entropy] + ([y.top_log_probs] if case["top"] else [])
            (grads,) = torch.autograd.grad(parts, (s["Z"],), s["C"])
        out = y
    result = dict(log_probs=[c.detach() for c in out.log_probs.coeffs], entropy=[c.detach() for c in out.entropy.coeffs])
    if case["top"]:
        result.update(top_tokens=out.top_tokens, top_log_probs=[c.detach() for c in out.top_log_probs.coeffs])
    if grads is not None:
        result["dz"] = list(grads.coeffs)
    return result


def _own_dropout(s):
    from polytensors_amd import PolyTensor

    if not s["case"]["grad"]:
        with torch.no_grad(), PolyTensor.plain_range():
            return dict(y=list(PolyTensor.dropout(s["X"], s["case"]["p"], seed=s["seed"]).coeffs))
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        y = PolyTensor.dropout(s["X"], s["case"]["p"], seed=s["seed"])
        (dx,) = torch.autograd.grad((y,), (s["X"],), (s["C"],))
        return dict(y=[c.detach() for c in y.coeffs], dx=list(dx.coeffs))


# ---------------------------------------------------------------------------
# Plain forms

def _acc(t):
    return t if t.dtype == torch.float64 else t.float()


def _conv(a, b):
    return [sum(a[i] * b[k - i] for i in range(k + 1)) for k in range(len(a))]


def _rsqrt(s):
    r = [torch.rsqrt(s[0])]
    for k in range(1, len(s)):
        r.append(-sum(((2 * k - i) / (2 * k)) * (s[i] / s[0]) * r[k - i] for i in range(1, k + 1)))
    return r


def _rotate(x, cos, sin, rotary, interleaved):
    """The first ``rotary`` elements of each head turned by the angles of its position (x: B, L, H, D)."""
    r, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((out, rest), -1)


def _plain_qk(s):
    case = s["case"]
    R, inter = case["rotary"], case["interleaved"]
    cos, sin = (s[n][s["positions"]][:, :, None, :] for n in ("cos", "sin"))
    out = {}
    for name in ("q", "k"):
        x, w = [_acc(c) for c in s[name]], _acc(s["w" + name])
        sq = [c.mean(-1, keepdim=True) for c in _conv(x, x)]
        sq[0] = sq[0] + EPS
        r = _rsqrt(sq)
        n = _conv(x, r)
        out[name] = [_rotate(c * w, cos, sin, R, inter).transpose(1, 2).contiguous().to(s[name][0].dtype) for c in n]
        if case["grad"]:   # the gradient of sum_k <cotangent_k, y_k>: the gradient series of the reversed cotangents, reversed
            g = [_rotate(_acc(c).transpose(1, 2), cos, -sin, R, inter) for c in s["c" + name][::-1]]
            out["dw" + name] = sum((a * b).sum((0, 1, 2)) for a, b in zip(n, g[::-1])).to(s["w" + name].dtype)
            gw = [c * w for c in g]
            u = [c.mean(-1, keepdim=True) for c in _conv(x, gw)]
            c3 = _conv(_conv(r, _conv(r, r)), u)
            dx = [a - b for a, b in zip(_conv(r, gw), _conv(c3, x))]
            out["d" + name] = [c.to(s[name][0].dtype) for c in dx[::-1]]
    return out


def _exp_series(z):
    """exp of a series (its constant order given by the exponential itself)."""
    e = [torch.exp(z[0])]
    for k in range(1, len(z)):
        e.append(sum((j / k) * z[j] * e[k - j] for j in range(1, k + 1)))
    return e


def _tanh_cap(z, cap):
    """cap tanh(z / cap) and its derivative series 1 - tanh^2."""
    u = [c / cap for c in z]
    y = [torch.tanh(u[0])]
    d = [1 - y[0] * y[0]]
    for k in range(1, len(z)):
        y.append(sum((j / k) * u[j] * d[k - j] for j in range(1, k + 1)))
        d.append(-sum(y[i] * y[k - i] for i in range(k + 1)))
    return [c * cap for c in y], d


def _plain_logprob(s):
    case = s["case"]
    K, top = case["degree"], case["top"]
    raw = [_acc(c) for c in s["z"]]
    z, slope = (raw, None) if case["softcap"] is None else _tanh_cap(raw, case["softcap"])
    keep = s["tokens"] != -100
    y = s["tokens"].clamp_min(0)[:, None]
    m = z[0].amax(1, keepdim=True)
    e = _exp_series([z[0] - m] + z[1:])
    total = [c.sum(1, keepdim=True) for c in e]
    nrm = [c / total[0] for c in total]
    lse = [m + total[0].log()]
    for k in range(1, K + 1):
        lse.append(nrm[k] - sum((i / k) * lse[i] * nrm[k - i] for i in range(1, k)))
    logp = [a - b for a, b in zip(z, lse)]
    p = _exp_series(logp)
    ent = [-c.sum(1) for c in _conv(p, logp)]
    zero = torch.zeros((), dtype=ent[0].dtype, device=ent[0].device)
    out = dict(log_probs=[torch.where(keep, c.gather(1, y)[:, 0], zero) for c in logp],
               entropy=[torch.where(keep, c, zero) for c in ent])
    if top:
        ids = torch.sort(raw[0], dim=1, descending=True, stable=True).indices[:, :top]
        if ids.shape[1] < top:
            raise ValueError("more alternatives than classes")
        out["top_tokens"] = torch.where(keep[:, None], ids, -1)
        out["top_log_probs"] = [torch.where(keep[:, None], c.gather(1, ids), zero) for c in logp]
    if case["grad"]:   # dz = -p (*) (c + ch (*) (log p + H)) + the cotangents at their tokens
        cl = [torch.where(keep, c, zero)[:, None] for c in s["cl"]]
        ch = [torch.where(keep, c, zero)[:, None] for c in s["ch"]]
        ct = [torch.where(keep[:, None], c, zero) for c in s["ct"]] if top else None
        c = cl if not top else [a + b.sum(1, keepdim=True) for a, b in zip(cl, ct)]
        inner = [a + b for a, b in zip(c, _conv(ch, [a + b[:, None] for a, b in zip(logp, ent)]))]
        dz = [-v for v in _conv(p, inner)]
        for k in range(K + 1):
            dz[k].scatter_add_(1, y, cl[k])
            if top:
                dz[k].scatter_add_(1, ids, ct[k])
        if slope is not None:
            dz = _conv(dz, slope)
        out["dz"] = [c.to(s["z"][0].dtype) for c in dz]
    return out


M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
LOW = 0xFFFFFFFF


def _plain_keep(seed, numel, p):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) over the counters 0, 1, ..: word i mod 4 of block i // 4 is
    element i's; it is kept where the word is at least p 2^32."""
    c = torch.arange((numel + 3) // 4, device=seed.device, dtype=torch.int64)
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    c0, c1, c2, c3 = c & LOW, (c >> 32) & LOW, torch.zeros_like(c), torch.zeros_like(c)

    def mul(a, m):   # the 64-bit product's halves: 64-bit products wrap, their bits do not care
        full = a * m
        return (full >> 32) & LOW, full & LOW

    for _ in range(10):
        h0, l0 = mul(c0, M0)
        h1, l1 = mul(c2, M1)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    return torch.stack((c0, c1, c2, c3), 1).flatten()[:numel] >= int(p * 2.0 ** 32)


def _plain_dropout(s):
    x, p = s["x"], s["case"]["p"]
    keep = _plain_keep(s["seed"], x[0].numel(), p).view(x[0].shape)

    def apply(series):
        return [(_acc(c) * (1.0 / (1.0 - p)) * keep).to(c.dtype) for c in series]

    out = dict(y=apply(x))
    if s["case"]["grad"]:
        out["dx"] = apply(s["c"])
    return out


# ---------------------------------------------------------------------------
# Work: each input read once and each output written once; the operations of the series rules

def work(case):
    K, e, grad = case["degree"], SIZES[case["dtype"]], case["grad"]
    n, pairs = K + 1, (K + 1) * (K + 2) // 2
    if case["kind"] == "qk":
        tokens = case["batch"] * case["length"]
        one = n * tokens * (case["heads"] + case["kv_heads"]) * case["head"]
        acc = 8 if case["dtype"] == "f64" else 4
        tables = min(case["table"], tokens) * case["rotary"] * acc + tokens * 8
        # squares, the product with the inverse root, the weight, the rotation; the gradient's four products
        return dict(bytes=e * one * (4 if grad else 2) + tables, flops=one / n * (4 * pairs + 4 * n) * (3 if grad else 1))
    if case["kind"] == "logprob":
        one = n * case["rows"] * case["classes"]
        acc = 8 if case["dtype"] == "f64" else 4
        small = case["rows"] * (8 + (2 + case["top"]) * n * acc * (2 if grad else 1) + 8 * case["top"])
        return dict(bytes=e * one * (2 if grad else 1) + small, flops=one / n * 4 * pairs * (3 if grad else 1))
    one = n * case["rows"] * case["width"]
    # a multiplication an element and order, and the generator: ten rounds of two products and four xors for four elements
    return dict(bytes=e * one * (4 if grad else 2), flops=one * (2 if grad else 1) + one / n * 20)


# ---------------------------------------------------------------------------
# 64-bit results

def _poly_mul(a, b):
    out = [torch.zeros_like(a[0] * b[0]) for _ in a]
    for i, x in enumerate(a):
        for j, y in enumerate(b):
            if i + j < len(out):
                out[i + j] = out[i + j] + x * y
    return out


def _poly_log(s):
    """t L' s = t s' solved for L."""
    out = [s[0].log()]
    for k in range(1, len(s)):
        v = k * s[k]
        for i in range(1, k):
            v = v - i * out[i] * s[k - i]
        out.append(v / (k * s[0]))
    return out


def _poly_exp(u):
    """exp as its power series in the part of u that vanishes at t = 0."""
    tail = [torch.zeros_like(u[0])] + list(u[1:])
    term = [torch.ones_like(u[0])] + [torch.zeros_like(u[0]) for _ in u[1:]]
    out = list(term)
    for j in range(1, len(u)):
        term = [c / j for c in _poly_mul(term, tail)]
        out = [a + b for a, b in zip(out, term)]
    return [u[0].exp() * c for c in out]


def _coefficient_grads(outputs, cotangents, leaves):
    return torch.autograd.grad([y for y in outputs], leaves, cotangents)


def _exact_qk(case, t):
    out = {}
    angle_cos, angle_sin = (t[n].double()[t["positions"]] for n in ("cos", "sin"))   # (B, L, R / 2)
    R = case["rotary"]
    index = torch.arange(R, device=DEV).view(-1, 2) if case["interleaved"] else torch.arange(R, device=DEV).view(2, -1).t()
    first, second = index[:, 0], index[:, 1]
    for name in ("q", "k"):
        x = [c.double().requires_grad_(case["grad"]) for c in t[name]]
        w = t["w" + name].double().requires_grad_(case["grad"])
        square = [c.mean(-1, keepdim=True) for c in _poly_mul(x, x)]
        square[0] = square[0] + EPS
        unit = _poly_mul(x, _poly_exp([-0.5 * c for c in _poly_log(square)]))
        turned = []
        for c in unit:
            v = (c * w).permute(0, 2, 1, 3)
            a, b = v[..., first], v[..., second]
            co, si = angle_cos[:, None], angle_sin[:, None]
            v = v.index_copy(3, first, a * co - b * si).index_copy(3, second, a * si + b * co)
            turned.append(v)
        out[name] = [c.detach() for c in turned]
        if case["grad"]:
            got = _coefficient_grads(turned, [c.double() for c in t["c" + name]], [*x, w])
            out["d" + name], out["dw" + name] = list(got[:-1]), got[-1]
    return out


def _exact_logprob_rows(case, z, tokens, cl, ch, ct):
    z = [c.double().requires_grad_(case["grad"]) for c in z]
    u = z
    if case["softcap"] is not None:   # tanh(v) = 1 - 2 / (exp(2 v) + 1)
        cap = case["softcap"]
        e = _poly_exp([2.0 * c / cap for c in z])
        inverse = _poly_exp([-c for c in _poly_log([e[0] + 1.0] + e[1:])])
        u = [cap * (1.0 - 2.0 * inverse[0])] + [-2.0 * cap * c for c in inverse[1:]]
    shift = u[0].detach().amax(1, keepdim=True)
    lse = _poly_log([c.sum(1, keepdim=True) for c in _poly_exp([u[0] - shift] + list(u[1:]))])
    lse[0] = lse[0] + shift
    logp = [a - b for a, b in zip(u, lse)]
    entropy = [-c.sum(1) for c in _poly_mul(_poly_exp(logp), logp)]
    keep = (tokens != -100).double()
    at = tokens.clamp_min(0)[:, None]
    out = dict(log_probs=[c.gather(1, at)[:, 0] * keep for c in logp], entropy=[c * keep for c in entropy])
    parts, cots = out["log_probs"] + out["entropy"], cl + ch
    if case["top"]:
        order = torch.sort(-z[0].detach(), dim=1, stable=True).indices[:, :case["top"]]
        out["top_tokens"] = torch.where(tokens[:, None] != -100, order, -1)
        out["top_log_probs"] = [c.gather(1, order) * keep[:, None] for c in logp]
        parts, cots = parts + out["top_log_probs"], cots + ct
    if case["grad"]:   # the gradient series J(x(t))^T c(t): reversed cotangents, read in reverse
        n = case["degree"] + 1
        flipped = [c for i in range(0, len(cots), n) for c in cots[i:i + n][::-1]]
        out["dz"] = list(_coefficient_grads(parts, [c.double() for c in flipped], z))[::-1]
    return {k: [c.detach() for c in v] if isinstance(v, list) else v for k, v in out.items()}


def _exact_logprob(case, t):
    N, C, n = case["rows"], case["classes"], case["degree"] + 1
    step = max(1, int(1.2e9) // (C * n * n * (4 if case["grad"] else 1)))   # rows at once: rows are independent
    parts = []
    for i in range(0, N, step):
        cut = lambda v: [c[i:i + step] for c in t[v]] if v in t else []   # noqa: E731
        parts.append(_exact_logprob_rows(case, cut("z"), t["tokens"][i:i + step], cut("cl"), cut("ch"), cut("ct")))
    return {k: [torch.cat([p[k][j] for p in parts]) for j in range(n)] if isinstance(parts[0][k], list)
            else torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_dropout(case, t):
    numel = t["x"][0].numel()
    seed = int(t["seed"].item()) % 2 ** 64
    mask = np.uint64(LOW)
    block = np.arange((numel + 3) // 4, dtype=np.uint64)
    word = [block & mask, block >> np.uint64(32), np.zeros_like(block), np.zeros_like(block)]
    for i in range(10):
        key = [np.uint64((seed % 2 ** 32 + i * W0) % 2 ** 32), np.uint64((seed // 2 ** 32 + i * W1) % 2 ** 32)]
        a, b = word[0] * np.uint64(M0), word[2] * np.uint64(M1)
        word = [(b >> np.uint64(32)) ^ word[1] ^ key[0], b & mask, (a >> np.uint64(32)) ^ word[3] ^ key[1], a & mask]
    keep = (np.stack(word, 1).reshape(-1)[:numel] >= np.uint64(int(case["p"] * 2.0 ** 32)))
    keep = torch.from_numpy(keep).to(DEV).view(t["x"][0].shape)
    out = {}
    for name, source in (("y", "x"), ("dx", "c")):
        if source in t:
            out[name] = [torch.where(keep, c.double() / (1.0 - case["p"]), 0.0) for c in t[source]]
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    return {"qk": _exact_qk, "logprob": _exact_logprob, "dropout": _exact_dropout}[case["kind"]](case, t)
