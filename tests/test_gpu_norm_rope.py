"""Per-head RMSNorm and rotation of series queries and keys against the definition in float64.

Tolerance, per order: half a rounding step of the storage type relative to each value, and rounding errors
of the arithmetic type (u = 2^-24, or 2^-53) relative to the order's largest value. A result is reached by at most
16 + 8 (K + 1)^2 roundings one after the other (a lane's and the lanes' row sums, the root series' K^2
terms, the products of K + 1 terms), and its terms sum to at most about 8 times the largest result for
coefficients that shrink by halves: 8 (16 + 8 (K + 1)^2) u. Gradients pass twice as many products; a weight's
also sums over rows, whose number (as a square root: errors of both signs) multiplies the bound.
Heads of one or two elements are another matter: x (mean x^2 + eps)^(-1/2) of a single element is its sign but
for eps, so that the terms of an order, each of the size of x_1 / x_0, cancel to about eps. There the scale
is not 8 times the result but twice (a rotation adds two elements) the sum of the terms' absolute values:
the same formulas with every product and sum taken of absolute values (``_majorants``).
"""

import math

import pytest
import torch

from polytensors_amd import PolyTensor
from tests import series64

pytestmark = pytest.mark.gpu

DTYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def _series(shape, degree, seed, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(shape, generator=g, dtype=torch.float64) * scale * 0.5 ** k).to(dtype) for k in range(degree + 1)]


def _tables(rows, rotary, dtype):
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, rotary, 2).double() / max(rotary, 1))
    return angle.cos().to(acc), angle.sin().to(acc)


def _bound(want, degree, dtype, factor=1.0, terms=None):
    u = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    step = 0.0 if dtype in (torch.float64, torch.float32) else torch.finfo(dtype).eps / 2
    scale = 8 * want.abs().max() if terms is None else 2 * terms.max()
    return want.abs() * step + factor * (16 + 8 * (degree + 1) ** 2) * u * scale


def _majorants(x, w, g, eps):
    """Sums of the terms' absolute values of y, of dx (g: coefficient cotangents, (B, H, L, D)) and of dw."""
    x, w, g = [c.double().abs() for c in x], w.double().abs(), [c.double().abs().transpose(1, 2) for c in g[::-1]]
    mean = lambda s: [c.mean(-1, keepdim=True) for c in s]   # noqa: E731
    s = mean(series64.mul(x, x))
    s[0] = s[0] + eps
    r = [s[0] ** -0.5]
    for k in range(1, len(s)):
        r.append(sum(((2 * k - i) / (2 * k)) * (s[i] / s[0]) * r[k - i] for i in range(1, k + 1)))
    n = series64.mul(x, r)
    h = [2 * c * w for c in g]
    c3 = series64.mul(series64.mul(r, series64.mul(r, r)), mean(series64.mul(x, h)))
    dx = [a + b for a, b in zip(series64.mul(r, h), series64.mul(c3, x))]
    return [c * w for c in n], dx[::-1], 2 * series64.mul(n, g)[-1].sum()


def _check(got, want, dtype, factor=1.0, what="", terms=None):
    degree = len(want) - 1
    for k, (a, b) in enumerate(zip(got, want)):
        assert a.shape == b.shape and a.dtype == dtype, (what, k, a.shape, b.shape)
        a, b = a.detach().cpu().double(), b.detach().double()
        bound = _bound(b, degree, dtype, factor, None if terms is None else terms[k])
        assert ((a - b).abs() <= bound).all(), f"{what} order {k}: {((a - b).abs() / bound.clamp_min(1e-300)).max():.3g} times the bound"


def _poly(cs):
    return PolyTensor(tuple(c.cuda() for c in cs))


def _double(cs):
    return None if cs is None else [c.double() for c in cs]


def _case(B, L, H, G, D, R, degree, dtype, weights="ordinary", seed=0, rows=None):
    q, k = _series((B, L, H, D), degree, seed + 1, dtype), _series((B, L, G, D), degree, seed + 2, dtype)
    n = 1 if weights == "ordinary" else degree + 1
    w = [None, None] if weights is None else \
        [[c + (1.0 if i == 0 else 0.0) for i, c in enumerate(_series((D,), n - 1, seed + 3 + j, dtype, 0.25))] for j in range(2)]
    cos, sin = _tables(rows or max(L, 8), R, dtype)
    return q, k, w, cos, sin


# (B, L, H, G, D, rotary, interleaved): one token, powers of two, heads of no power of two, a part rotated,
# nothing rotated, odd heads, single elements, the largest head, lengths off the blocks
SHAPES = [(3, 1, 8, 2, 128, 128, False), (1, 1, 1, 1, 64, 64, True), (2, 5, 4, 4, 64, 32, False), (2, 7, 3, 1, 80, 20, True),
          (1, 33, 2, 2, 96, 96, False), (2, 3, 2, 1, 17, 16, False), (2, 3, 2, 1, 17, 8, True), (1, 9, 3, 3, 256, 256, False),
          (1, 4, 2, 2, 1, 0, False), (1, 4, 2, 2, 2, 2, True), (2, 6, 2, 2, 130, 6, False), (1, 5, 1, 1, 255, 254, True),
          (2, 65, 5, 2, 32, 0, False), (1, 3, 1, 1, 40, 12, False), (1, 8, 16, 2, 192, 64, True)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_and_coefficient_gradients(shape, dtype):
    B, L, H, G, D, R, interleaved = shape
    for degree in (1, 3):
        q, k, w, cos, sin = _case(B, L, H, G, D, R, degree, dtype, seed=10 * degree)
        positions = torch.randint(0, cos.shape[0], (B, L), generator=torch.Generator().manual_seed(3))
        cq, ck = _series((B, H, L, D), degree, 7, dtype), _series((B, G, L, D), degree, 8, dtype)
        leaves = [c.cuda().requires_grad_() for c in (*q, *k, w[0][0], w[1][0])]
        n = degree + 1
        with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
            yq, yk = PolyTensor.qk_norm_rope(PolyTensor(tuple(leaves[:n])), PolyTensor(tuple(leaves[n:2 * n])), cos.cuda(),
                                             sin.cuda(), positions.cuda(), leaves[-2], leaves[-1], 1e-5, interleaved)
        grads = torch.autograd.grad((*yq.coeffs, *yk.coeffs), leaves, [c.cuda() for c in (*cq, *ck)])
        with torch.no_grad(), PolyTensor.plain_range():   # without a graph: the stacked form
            plain = PolyTensor.qk_norm_rope(_poly(q), _poly(k), cos.cuda(), sin.cuda(), positions.cuda(), w[0][0].cuda(),
                                            w[1][0].cuda(), 1e-5, interleaved)
        for got, stacked in zip((yq, yk), plain):
            assert all(torch.equal(a, b) for a, b in zip(got.coeffs, stacked.coeffs))
        factor = 2 * math.sqrt(B * L * max(H, G))
        for y, x, weight, c, d in ((yq, q, w[0], cq, (*grads[:n], grads[-2])), (yk, k, w[1], ck, (*grads[n:2 * n], grads[-1]))):
            x64 = [t.double().requires_grad_() for t in x]
            w64 = [weight[0].double().requires_grad_()]
            want = series64.norm_rope(x64, w64, cos.double(), sin.double(), positions, 1e-5, interleaved)
            y_terms, dx_terms, dw_terms = _majorants(x, weight[0], c, 1e-5) if D <= 2 else (None, None, None)
            _check(y.coeffs, want, dtype, 1, "y", y_terms)
            ref = torch.autograd.grad(want, x64 + w64, _double(c))
            _check(d[:-1], list(ref[:-1]), dtype, 2, "dx", dx_terms)
            _check([d[-1]], [ref[-1]], dtype, factor * (degree + 1) ** 2, "dw", None if D > 2 else [dw_terms])


@pytest.mark.parametrize("degree", range(9))
@pytest.mark.parametrize("D,R,interleaved", [(64, 64, False), (64, 32, True), (33, 10, False)])
@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_every_degree_with_series_weights_and_wrapper_gradients(degree, D, R, interleaved, dtype):
    q, k, w, cos, sin = _case(2, 5, 3, 2, D, R, degree, dtype, weights="series", seed=degree)
    cq, ck = _series((2, 3, 5, D), degree, 7, dtype), _series((2, 2, 5, D), degree, 8, dtype)
    inputs = [PolyTensor(tuple(c.cuda() for c in s), requires_grad=True) for s in (q, k, w[0], w[1])]
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        yq, yk = PolyTensor.qk_norm_rope(inputs[0], inputs[1], cos.cuda(), sin.cuda(), None, inputs[2], inputs[3], 1e-4,
                                         interleaved)
        grads = torch.autograd.grad((yq, yk), inputs, (_poly(cq), _poly(ck)))
        positions = torch.arange(5).expand(2, 5)
        for y, x, weight, c, dx, dw in ((yq, q, w[0], cq, grads[0], grads[2]), (yk, k, w[1], ck, grads[1], grads[3])):
            x64, w64 = [t.double().requires_grad_() for t in x], [t.double().requires_grad_() for t in weight]
            want = series64.norm_rope(x64, w64, cos.double(), sin.double(), positions, 1e-4, interleaved)
            _check(y.coeffs, want, dtype, what="y")
            # the gradient series: coefficient gradients of the reversed cotangents, reversed
            ref = torch.autograd.grad(want, x64 + w64, _double(c[::-1]))
            _check(dx.coeffs, list(ref[:degree + 1])[::-1], dtype, 2, "dx")
            _check(dw.coeffs, list(ref[degree + 1:])[::-1], dtype, 2 * math.sqrt(30), "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_a_projection_and_other_strides(dtype):
    B, L, H, D, degree = 2, 6, 3, 64, 2
    rows = _series((B, L, 3 * H * D), degree, 5, dtype)
    cos, sin = _tables(L, 64, dtype)
    positions = torch.arange(L).expand(B, L)
    views = {
        "projection": lambda r: (r.view(B, L, 3 * H, D)[:, :, :H], r.view(B, L, 3 * H, D)[:, :, H:2 * H]),
        "odd offset": lambda r: (r.flatten()[3:3 + B * L * H * D].view(B, L, H, D), r.view(B, L, 3 * H, D)[:, :, 1:2]),
        "heads first": lambda r: (r.view(B, 3 * H, L, D).transpose(1, 2), r.view(B, L, 3 * H, D)),
        "element stride": lambda r: (r.view(B, L, D, 3 * H).transpose(2, 3)[:, :, :H], r.view(B, L, 3 * H, D).flip(3)),
        "expanded": lambda r: (r.view(B, L, 3 * H, D)[:, :, :1].expand(B, L, H, D), r.view(B, L, 3 * H, D)[:1].expand(B, -1, -1, -1)),
    }
    for name, view in views.items():
        parts = [view(r) for r in rows]
        cuda = [view(r.cuda()) for r in rows]
        q, k = PolyTensor._wrap(tuple(c[0] for c in cuda)), PolyTensor._wrap(tuple(c[1] for c in cuda))
        with torch.no_grad(), PolyTensor.plain_range():
            yq, yk = PolyTensor.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), eps=1e-5)
        for i, y in enumerate((yq, yk)):
            assert all(c.is_contiguous() for c in y.coeffs)
            want = series64.norm_rope([p[i].double() for p in parts], None, cos.double(), sin.double(), positions, 1e-5, False)
            _check(y.coeffs, want, dtype, what=name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_and_positions_without_an_angle(dtype):
    B, L, H, G, D, degree = 3, 4, 2, 1, 64, 2
    q, k, w, cos, sin = _case(B, L, H, G, D, D, degree, dtype, rows=6)
    positions = torch.tensor([[0, 1, 2, 3], [4, 5, -1, -1], [-5, 6, 2, -2 ** 62]])   # 6: past the table
    for c in (*q, *k):   # whatever padding holds stays out of results and gradients
        c[positions < 0] = float("nan")
    leaves = [c.cuda().requires_grad_() for c in (*q, *k, w[0][0], w[1][0])]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        outs = PolyTensor.qk_norm_rope(PolyTensor(tuple(leaves[:3])), PolyTensor(tuple(leaves[3:6])), cos.cuda(), sin.cuda(),
                                       positions.cuda(), leaves[6], leaves[7], 1e-5)
    coeffs = [c for y in outs for c in y.coeffs]
    for c in coeffs:
        by_token = c.detach().cpu().transpose(1, 2)
        assert not by_token[positions < 0].any() and by_token[positions == 6].isnan().all()
        assert by_token[(positions >= 0) & (positions < 6)].isfinite().all()
    cots = [torch.ones_like(c) for c in coeffs]
    grads = torch.autograd.grad(coeffs, leaves, cots)
    for g in grads[:6]:
        g = g.cpu()
        assert not g[positions < 0].any() and g[positions == 6].isnan().all()
        assert g[(positions >= 0) & (positions < 6)].isfinite().all()
    # without the row past the table the weights' gradients are finite: padding adds nothing
    positions[2, 1] = -1
    for c in (*leaves[:6],):
        c.data[2, 1] = float("nan")
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        outs = PolyTensor.qk_norm_rope(PolyTensor(tuple(leaves[:3])), PolyTensor(tuple(leaves[3:6])), cos.cuda(), sin.cuda(),
                                       positions.cuda(), leaves[6], leaves[7], 1e-5)
    grads = torch.autograd.grad([c for y in outs for c in y.coeffs], leaves[6:], cots)
    keep = positions >= 0
    for x, weight, g in ((q, w[0], grads[0]), (k, w[1], grads[1])):
        x64, w64 = [torch.where(keep[..., None, None], c.double(), 0.0) for c in x], weight[0].double().requires_grad_()
        want = series64.norm_rope(x64, [w64], cos.double(), sin.double(), positions, 1e-5, False)
        (ref,) = torch.autograd.grad(want, [w64], [torch.ones_like(c) for c in want])
        _check([g], [ref], dtype, 2 * math.sqrt(24) * 9, "dw")


def test_zero_rows_and_eps():
    D = 32
    cos, sin = _tables(8, D, torch.float32)
    x = torch.zeros(1, 2, 1, D)
    x[0, 1] = 3.0
    zero = PolyTensor((x.cuda(), torch.ones_like(x).cuda()))
    with torch.no_grad(), PolyTensor.plain_range():
        y, _ = PolyTensor.qk_norm_rope(zero, zero, cos.cuda(), sin.cuda(), eps=1e-2)
        want = series64.norm_rope([x.double(), torch.ones_like(x).double()], None, cos.double(), sin.double(),
                                  torch.arange(2)[None], 1e-2, False)
        _check(y.coeffs, want, torch.float32)
        default, _ = PolyTensor.qk_norm_rope(zero, zero, cos.cuda(), sin.cuda())
        same, _ = PolyTensor.qk_norm_rope(zero, zero, cos.cuda(), sin.cuda(), eps=torch.finfo(torch.float32).eps)
    assert all(torch.equal(a, b) for a, b in zip(default.coeffs, same.coeffs))


def test_an_ordinary_operand_and_a_single_gradient():
    q, k, w, cos, sin = _case(2, 3, 2, 2, 64, 64, 2, torch.float64)
    positions = torch.arange(3).expand(2, 3)
    with torch.no_grad(), PolyTensor.plain_range():
        yq, yk = PolyTensor.qk_norm_rope(_poly(q), k[0].cuda(), cos.cuda(), sin.cuda(), key_weight=w[1][0].cuda(), eps=1e-5)
    assert isinstance(yq, PolyTensor) and type(yk) is torch.Tensor
    _check(yq.coeffs, series64.norm_rope(q, None, cos, sin, positions, 1e-5, False), torch.float64)
    _check([yk], series64.norm_rope(k[:1], w[1], cos, sin, positions, 1e-5, False), torch.float64)
    with torch.no_grad(), PolyTensor.plain_range():   # an ordinary operand under a series weight is a series
        _, yk = PolyTensor.qk_norm_rope(_poly(q), k[0].cuda(), cos.cuda(), sin.cuda(), key_weight=_poly(q[0:3])[0, 0, 0], eps=1e-5)
    assert yk.degree == 2
    # only the keys' gradient asked for, and only the queries' output used
    x, z = PolyTensor(tuple(c.cuda() for c in q), requires_grad=True), PolyTensor(tuple(c.cuda() for c in k), requires_grad=True)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        yq, yk = PolyTensor.qk_norm_rope(x, z, cos.cuda(), sin.cuda(), eps=1e-5)
        c = _series((2, 2, 3, 64), 2, 9, torch.float64)
        (dz,) = torch.autograd.grad((yk,), (z,), (_poly(c),), retain_graph=True)
        dx, none = torch.autograd.grad((yq,), (x, z), (_poly(c),), allow_unused=True)
        assert none is None
        for x64, d in ((k, dz), (q, dx)):
            x64 = [t.double().requires_grad_() for t in x64]
            ref = torch.autograd.grad(series64.norm_rope(x64, None, cos, sin, positions, 1e-5, False), x64, c[::-1])
            _check(d.coeffs, list(ref)[::-1], torch.float64, 2)


def test_gradient_against_differences():
    q, k, w, cos, sin = _case(1, 3, 1, 1, 10, 6, 2, torch.float64)
    c = _series((1, 1, 3, 10), 2, 4, torch.float64)

    def value(q, w):
        with torch.no_grad(), PolyTensor.plain_range():
            y, _ = PolyTensor.qk_norm_rope(_poly(q), _poly(k), cos.cuda(), sin.cuda(), None, w.cuda(), None, 1e-3)
        return sum((a.cpu() * b).sum() for a, b in zip(y.coeffs, c)).item()

    leaves = [t.cuda().requires_grad_() for t in (*q, w[0][0])]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y, _ = PolyTensor.qk_norm_rope(PolyTensor(tuple(leaves[:3])), _poly(k), cos.cuda(), sin.cuda(), None, leaves[3], None, 1e-3)
    grads = torch.autograd.grad(y.coeffs, leaves, [t.cuda() for t in c])
    h = 1e-5   # central differences: error h^2 times third derivatives of order one, and rounding 2^-53 / h
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        moved = lambda s: value([x + s * d if j == i else x for j, x in enumerate(q)], w[0][0] + (s * d if i == 3 else 0))   # noqa: E731
        slope = (moved(h) - moved(-h)) / (2 * h)
        got = (grads[i].cpu() * d).sum().item()
        assert abs(slope - got) <= 1e-7 * max(1.0, abs(got)), i


def test_complex_directions():
    base, real, imag = _series((2, 3, 2, 32), 2, 1, torch.float64)
    cos, sin = _tables(3, 32, torch.float64)
    x = [base, torch.complex(real, imag), torch.complex(imag, real)]
    with torch.no_grad(), PolyTensor.plain_range():
        yq, yk = PolyTensor.qk_norm_rope(_poly(x), _poly([base, real, imag]), cos.cuda(), sin.cuda(), eps=1e-4)
    want = series64.norm_rope([c.to(torch.complex128) for c in x], None, cos, sin, torch.arange(3).expand(2, 3), 1e-4, False)
    for k in range(3):
        got = yq.coeffs[k].cpu()
        assert (got - (want[k].real if k == 0 else want[k])).abs().max() <= 1e-12
    assert not yk.coeffs[1].is_complex()


def test_complex_directions_in_reverse_mode():
    # the gradient series along a complex direction: the real definition's, extended to complex coefficients
    base, real, imag = _series((1, 2, 1, 16), 2, 3, torch.float64)
    cot = _series((1, 1, 2, 16), 2, 4, torch.float64)
    cos, sin = _tables(2, 16, torch.float64)
    w = [c + (1.0 if i == 0 else 0.0) for i, c in enumerate(_series((16,), 2, 5, torch.float64, 0.2))]
    x = [base, torch.complex(real, imag), torch.complex(imag, real)]
    X, W = PolyTensor(tuple(c.cuda() for c in x), requires_grad=True), PolyTensor(tuple(c.cuda() for c in w), requires_grad=True)
    key = PolyTensor(tuple(c.cuda() for c in (base, real, imag)))
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        y, _ = PolyTensor.qk_norm_rope(X, key, cos.cuda(), sin.cuda(), query_weight=W, eps=1e-3)
        y.backward(_poly(cot))
        # d/dx_0 of <cotangents, y> for real series is coefficient K of the gradient series; polynomial in the
        # directions, so its value at complex ones comes from autograd over the complex definition
        z = [c.to(torch.complex128).requires_grad_() for c in x]
        v = [c.to(torch.complex128).requires_grad_() for c in w]
        want = series64.norm_rope(z, v, cos, sin, torch.arange(2)[None], 1e-3, False)
        total = sum((a * b).sum() for a, b in zip(want, cot[::-1]))
        ref = torch.autograd.grad(total.real, z + v, retain_graph=True)
        for i in range(3):   # (torch's gradient of the real part of a holomorphic function is the derivative's conjugate)
            for got, r in ((X.grad, ref[2 - i].conj()), (W.grad, ref[5 - i].conj())):
                got = got.coeffs[i].cpu().to(torch.complex128)
                assert (got - (r.real if i == 0 else r)).abs().max() <= 1e-9 * max(1.0, r.abs().max().item()), i


def test_gradients_of_nothing():
    cos, sin = _tables(4, 16, torch.float32)
    for B, L in ((0, 3), (2, 0)):
        leaf = torch.empty(B, L, 2, 16, device="cuda", requires_grad=True)
        w = torch.ones(16, device="cuda", requires_grad=True)
        with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
            x = PolyTensor((leaf,))
            y, z = PolyTensor.qk_norm_rope(x, x, cos.cuda(), sin.cuda(), None, w, None)
        dx, dw = torch.autograd.grad((y.value, z.value), (leaf, w), (torch.ones_like(y.value), torch.ones_like(z.value)))
        assert dx.shape == leaf.shape and not dw.any()


def test_another_stream():
    q, k, w, cos, sin = _case(2, 40, 4, 2, 64, 64, 1, torch.float32)
    stream = torch.cuda.Stream()
    Q, K = _poly(q), _poly(k)
    tables = cos.cuda(), sin.cuda()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.no_grad(), PolyTensor.plain_range():
        y, _ = PolyTensor.qk_norm_rope(Q, K, *tables, eps=1e-5)
    stream.synchronize()
    _check(y.coeffs, series64.norm_rope(_double(q), None, cos.double(), sin.double(), torch.arange(40).expand(2, 40), 1e-5, False),
           torch.float32)


def test_captured_training_step():
    q, k, w, cos, sin = _case(2, 9, 4, 2, 64, 64, 2, torch.bfloat16)
    leaves = [c.cuda().requires_grad_() for c in (*q, *k, w[0][0], w[1][0])]
    tables = cos.cuda(), sin.cuda()
    positions = torch.arange(9, device="cuda").repeat(2, 1)
    cots = [c.cuda() for c in (*_series((2, 4, 9, 64), 2, 7, torch.bfloat16), *_series((2, 2, 9, 64), 2, 8, torch.bfloat16))]

    def step():
        with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
            yq, yk = PolyTensor.qk_norm_rope(PolyTensor(tuple(leaves[:3])), PolyTensor(tuple(leaves[3:6])), *tables, positions,
                                             leaves[6], leaves[7], 1e-5)
        return torch.autograd.grad((*yq.coeffs, *yk.coeffs), leaves, cots)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for scale in (1.0, 0.5, 1.0):
        cots[0].mul_(scale)
        positions.add_(1).remainder_(8)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):   # the kernels have no order of their own to vary: bit for bit
            assert torch.equal(a, b)


def test_more_elements_than_32_bits_count():
    B, L, H, D = 1, 2 ** 20 + 1, 16, 128   # 2^31 + 2^11 elements
    x = torch.empty(B, L, H, D, dtype=torch.bfloat16, device="cuda").normal_()
    cos, sin = _tables(4, D, torch.bfloat16)
    positions = (torch.arange(L, device="cuda") % 4)
    small = torch.ones(B, L, 1, D, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad(), PolyTensor.plain_range():
        y, _ = PolyTensor.qk_norm_rope(PolyTensor((x,)), PolyTensor((small,)), cos.cuda(), sin.cuda(), positions, eps=1e-5)
        dx = torch.ops.polytensors_amd.norm_rope_series_backward([x], [], [y.value], [], cos.cuda(), sin.cuda(), positions, [], [],
                                                                 1e-5, False, 0, 0)[0][0]
    for part in (slice(0, 3), slice(L - 3, L)):
        x64 = [x[:, part].cpu().double().requires_grad_()]
        want = series64.norm_rope(x64, None, cos.double(), sin.double(), positions[part].cpu()[None], 1e-5, False)
        got = y.value[:, :, part].cpu()
        _check([got], want, torch.bfloat16)
        (ref,) = torch.autograd.grad(want, x64, [got.double()])
        # (the gradient along y itself nearly cancels: relative to the terms, of the size of y / |x|)
        assert (dx[:, part].cpu().double() - ref).abs().max() <= 2.0 ** -8 * ref.abs().max() + 3000 * 2.0 ** -24 * got.abs().max()


def test_refused_calls():
    q, k, w, cos, sin = _case(2, 3, 2, 1, 64, 64, 1, torch.float32)
    Q, K, c, s = _poly(q), _poly(k), cos.cuda(), sin.cuda()
    wq = w[0][0].cuda()
    bad = [
        ((Q, K, c.double(), s.double()), {}, "cos and sin"), ((Q, K, cos, sin), {}, "cos and sin"),
        ((Q, K, c[:, :1], s), {}, "cos and sin"), ((Q, K, torch.cat((c, c), 1), torch.cat((s, s), 1)), {}, "rotary"),
        ((Q, K[:, :2], c, s), {}, "must be"), ((Q[0], K[0], c, s), {}, "must be"), ((Q, K[..., :32], c, s), {}, "must be"),
        ((Q, K, c, s), dict(positions=torch.arange(3)), "positions"), ((Q, K, c, s), dict(positions=torch.arange(4).cuda()), "positions"),
        ((Q, K, c, s), dict(positions=torch.arange(3.0).cuda()), "positions"),
        ((Q, K, c, s), dict(query_weight=wq[:32]), "weights"), ((Q, K, c, s), dict(query_weight=wq.double()), "dtype"),
        ((Q, K, c, s), dict(eps=-1.0), "eps"), ((Q, K, c, s), dict(eps=float("nan")), "eps"),
        ((q[0].cuda(), k[0].cuda(), c, s), {}, "no PolyTensor"), ((Q, None, c, s), {}, "tensors"),
        ((Q, PolyTensor(tuple(t.cuda() for t in k), degree=2), c, s), {}, "degree"),
        ((PolyTensor((q[0].cuda(),), degree=9), PolyTensor((k[0].cuda(),), degree=9), c, s), {}, "degree 9"),
        ((_poly([torch.ones(1, 1, 1, 257)]), _poly([torch.ones(1, 1, 1, 257)]), c, s), {}, "256"),
    ]
    with torch.no_grad(), PolyTensor.plain_range():
        for args, kwargs, needle in bad:
            with pytest.raises(NotImplementedError, match=needle):
                PolyTensor.qk_norm_rope(*args, **kwargs)
        for B, L in ((0, 3), (2, 0)):   # nothing to do
            e = PolyTensor((torch.empty(B, L, 2, 64, device="cuda"),))
            y, z = PolyTensor.qk_norm_rope(e, e, c, s)
            assert y.shape == (B, 2, L, 64) and z.shape == (B, 2, L, 64)
    with PolyTensor.plain_range():
        X = PolyTensor(tuple(t.cuda() for t in q), requires_grad=True)
        with pytest.raises(NotImplementedError, match="ordinary"):
            PolyTensor.qk_norm_rope(X, K, c, s, query_weight=wq.clone().requires_grad_())
        with pytest.raises(NotImplementedError, match="tables"):
            with PolyTensor.coefficient_autograd():
                PolyTensor.qk_norm_rope(Q, K, c.clone().requires_grad_(), s)
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        leaf = [t.cuda().requires_grad_() for t in q]
        y, _ = PolyTensor.qk_norm_rope(PolyTensor(tuple(leaf)), K, c, s)
        with pytest.raises(NotImplementedError, match="second-order"):
            torch.autograd.grad(y.coeffs[0].sum(), leaf[0], create_graph=True)
