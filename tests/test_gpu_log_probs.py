"""Log probabilities, entropies and alternatives of series logits on the GPU against the definition in float64.

Tolerances, with u = 2^-24 (2^-53 in float64) and an order's scale max(1, its largest value): a thread adds
C / 256 classes and its sums meet in a tree; each exponential is off by up to |z - m| u (below 40 u here) and a
few units, the series rules add at most 8 (K + 1)^2 roundings of terms within 8 times the scale:
8 (C / 256 + 64 + 8 (K + 1)^2) u. The gradient is a product of such series, twice that, after half a
rounding step of its type. Classes chosen are whole numbers and must be equal.
"""

import pytest
import torch

from polytensors_amd import PolyTensor
from tests import series64

pytestmark = pytest.mark.gpu

DTYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def _series(shape, degree, seed, dtype, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(shape, generator=g, dtype=torch.float64) * scale * 0.5 ** k).to(dtype) for k in range(degree + 1)]


def _tokens(rows, classes, seed, ignored=True):
    t = torch.randint(0, classes, (rows,), generator=torch.Generator().manual_seed(seed))
    if ignored and rows > 2:
        t[1] = -100
    return t


def _poly(cs):
    return PolyTensor(tuple(c.cuda() for c in cs))


def _bound(degree, classes, dtype, want):
    u = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    return 8 * (classes / 256 + 64 + 8 * (degree + 1) ** 2) * u * max(1.0, want.abs().max().item())


def _check(got, want, classes, dtype, what):
    degree = len(want) - 1
    for k, (a, b) in enumerate(zip(got, want)):
        assert a.shape == b.shape and a.dtype == (torch.float64 if dtype == torch.float64 else torch.float32), what
        a, b = a.detach().cpu().double(), b.detach()
        finite = b.isfinite()
        assert torch.equal(a[~finite], b[~finite]), (what, k)
        a, b = a[finite], b[finite]
        if b.numel():
            bound = _bound(degree, classes, dtype, b)
            assert (a - b).abs().max() <= bound, f"{what} order {k}: {(a - b).abs().max():.3g} above {bound:.3g}"


def _check_gradient(got, want, classes, dtype, what="dz"):
    degree = len(want) - 1
    step = 0.0 if dtype in (torch.float64, torch.float32) else torch.finfo(dtype).eps / 2
    tiny = 0.0 if dtype == torch.float64 else 2.0 ** -25 if dtype == torch.float16 else 0.0   # half of float16's least step
    for k, (a, b) in enumerate(zip(got, want)):
        assert a.shape == b.shape and a.dtype == dtype
        a, b = a.detach().cpu().double(), b.detach()
        bound = b.abs() * step + tiny + 2 * _bound(degree, classes, dtype, b)
        assert ((a - b).abs() <= bound).all(), f"{what} order {k}: {((a - b).abs() / bound).max():.3g} times the bound"


def _run(Z, tokens, **kwargs):
    with torch.no_grad(), PolyTensor.plain_range():
        return PolyTensor.token_log_probs(_poly(Z), tokens.cuda(), **kwargs)


def _compare(Z, tokens, dtype, classes, **kwargs):
    got = _run(Z, tokens, **kwargs)
    want = series64.log_probs([c.double() for c in Z], tokens, **kwargs)
    _check(got.log_probs.coeffs, want[0], classes, dtype, "log_probs")
    _check(got.entropy.coeffs, want[1], classes, dtype, "entropy")
    if kwargs.get("top"):
        assert torch.equal(got.top_tokens.cpu(), want[2])
        _check(got.top_log_probs.coeffs, want[3], classes, dtype, "top_log_probs")
    else:
        assert got.top_tokens is None and got.top_log_probs is None
    return got


# rows, classes: one class, fewer than a vector, off the vectors, more than a block's threads, many vectors;
# few rows (cut into pieces) and many
SHAPES = [(1, 1), (3, 2), (5, 7), (4, 33), (2, 255), (3, 1000), (1, 4099), (2, 20011), (9, 8192), (1, 65537), (1100, 515), (1025, 64)]


@pytest.mark.parametrize("rows,classes", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(rows, classes, dtype):
    for degree, top in ((1, min(5, classes)), (3, 0)):
        _compare(_series((rows, classes), degree, rows + classes, dtype), _tokens(rows, classes, 1), dtype, classes, top=top)


@pytest.mark.parametrize("degree", range(9))
@pytest.mark.parametrize("softcap", [None, 4.0])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
def test_every_degree_and_softcap(degree, softcap, dtype):
    for rows, classes in ((6, 777), (2, 9001)):
        _compare(_series((rows, classes), degree, degree, dtype), _tokens(rows, classes, 2), dtype, classes, top=4, softcap=softcap)


@pytest.mark.parametrize("top", [1, 2, 3, 20, 31, 32])
@pytest.mark.parametrize("rows,classes", [(3, 32), (2, 100), (2, 6000), (1, 70001)])
def test_alternatives(top, rows, classes):
    for dtype in (torch.float32, torch.bfloat16):   # bfloat16: many equal logits
        _compare(_series((rows, classes), 1, top, dtype), _tokens(rows, classes, 3), dtype, classes, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_of_rows_arranged_against_them(dtype):
    top = 20
    for C in (40, 5000, 40000):
        g = torch.Generator().manual_seed(C)
        sorted_rows = torch.linspace(-4, 4, C, dtype=torch.float64)
        rows = [torch.zeros(C).double(), sorted_rows, sorted_rows.flip(0), torch.randint(0, 3, (C,), generator=g).double(),
                torch.where(torch.arange(C) % 256 == 7, 5.0, 0.0).double(),        # one thread holds the largest
                torch.where(torch.arange(C) % 2048 < 16, sorted_rows + 9, 0.0), -torch.zeros(C).double(),
                torch.where(torch.arange(C) % 2 == 0, -0.0, 0.0).double()]
        z0 = torch.stack(rows).to(dtype)
        Z = [z0, torch.randn(z0.shape, generator=g).to(dtype)]
        # (equal, and equally spaced, logits repeat a rounding of the sums: the log of C against C equal terms)
        _compare(Z, torch.arange(8), dtype, C, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [50, 9000])
def test_masked_classes_and_numbers_that_are_none(dtype, classes):
    rows, top = 6, 4
    Z = _series((rows, classes), 2, 5, dtype)
    tokens = _tokens(rows, classes, 6, ignored=False)
    Z[0][0, ::2] = -INF                      # masked: whatever the higher orders hold
    Z[1][0, ::2], Z[2][0, ::2] = float("nan"), INF
    Z[0][1, 3:] = -INF                       # three classes left: fewer than the alternatives
    Z[0][2, 1:] = -INF                       # one
    Z[0][3, ::3] = torch.finfo(dtype).min    # a mask of the type's lowest value
    tokens[:4] = torch.tensor([1, 2, 0, 1])
    got = _compare(Z, tokens, dtype, classes, top=top)
    assert got.log_probs.value[2].item() == 0.0 and abs(got.entropy.value[2].item()) < 1e-6
    # a masked token has probability zero; its higher orders are the shifted logits'
    tokens[1] = 7
    Z[1][1, 7] = 0.25
    again = _run(Z, tokens, top=top)
    assert again.log_probs.value[1].item() == -INF and again.log_probs.coeffs[1][1].isfinite()
    # rows without a distribution: no class left, an infinite or undefined logit
    for bad in (-INF, INF, float("nan")):
        Y = [c.clone() for c in Z]
        Y[0][4, :] = bad if bad == -INF else Y[0][4, :]
        Y[0][4, 11] = bad
        y = _run(Y, tokens, top=top)
        for c in (*y.log_probs.coeffs, *y.entropy.coeffs):
            assert c[4].isnan() and c[5].isfinite()
        want = torch.sort(Y[0].double(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(y.top_tokens.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_large_shifts_cost_no_digits(dtype):
    Z = _series((3, 2000), 2, 8, dtype)
    shift = 1024.0   # a power of two: adding it to values rounded to 2^-12 is exact
    Z = [(c * 4096).round() / 4096 for c in Z]
    tokens = _tokens(3, 2000, 9)
    # against the definition without the shift, which is the same, within the bound of values without it (with
    # the shift float64 itself loses digits in the plain definition)
    _compare(Z, tokens, dtype, 2000, top=3)
    got = _run([c + shift for c in Z], tokens, top=3)
    want = series64.log_probs([c.double() for c in Z], tokens, top=3)
    for a, b in ((got.log_probs, want[0]), (got.entropy, want[1]), (got.top_log_probs, want[3])):
        _check(a.coeffs, b, 2000, dtype, "shifted")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes", [(7, 33), (3, 4100), (300, 130), (1, 20011)])
@pytest.mark.parametrize("softcap", [None, 5.0])
def test_gradients(dtype, rows, classes, softcap):
    degree, top = 2, 6
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    Z, tokens = _series((rows, classes), degree, 11, dtype), _tokens(rows, classes, 12)
    cots = [_series((rows,), degree, 13, acc, 1.0), _series((rows,), degree, 14, acc, 0.5), _series((rows, top), degree, 15, acc, 0.5)]
    # the most probable class is a given token's too, in a few rows
    best = Z[0].double().argmax(1)
    tokens[2:4] = best[2:4]
    z64 = [c.double().requires_grad_() for c in Z]
    want = series64.log_probs(z64, tokens, top=top, softcap=softcap)
    parts = [want[0], want[1], want[3]]
    for use in ((0,), (1,), (2,), (0, 1), (0, 1, 2)):
        outs = [c for i in use for c in parts[i]]
        ref = torch.autograd.grad(outs, z64, [c.double() for i in use for c in cots[i]], retain_graph=True)
        leaves = [c.cuda().requires_grad_() for c in Z]
        with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
            y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), tokens.cuda(), top=top, softcap=softcap)
        mine = [y.log_probs, y.entropy, y.top_log_probs]
        got = torch.autograd.grad([c for i in use for c in mine[i].coeffs], leaves, [c.cuda() for i in use for c in cots[i]])
        _check_gradient(got, list(ref), classes, dtype)
        # the gradient series: reversed cotangents, reversed
        ref = torch.autograd.grad(outs, z64, [c.double() for i in use for c in cots[i][::-1]], retain_graph=True)[::-1]
        z = PolyTensor(tuple(c.cuda() for c in Z), requires_grad=True)
        with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
            y = PolyTensor.token_log_probs(z, tokens.cuda(), top=top, softcap=softcap)
            mine = [y.log_probs, y.entropy, y.top_log_probs]
            (got,) = torch.autograd.grad([mine[i] for i in use], (z,), [_poly(cots[i]) for i in use])
            _check_gradient(got.coeffs, list(ref), classes, dtype)


def test_gradients_of_masked_padded_and_undefined_rows():
    classes, dtype = 300, torch.float32
    Z, tokens = _series((4, classes), 2, 16, dtype), torch.tensor([4, -100, 7, classes + 3])
    Z[0][0, ::2] = -INF
    Z[1][0, ::2], Z[2][0, ::2] = float("nan"), -INF
    Z[0][1] = float("nan")    # padding holds anything
    Z[0][0, 4] = 1.0
    Z[1][0, 4] = Z[2][0, 4] = 0.5
    leaves = [c.cuda().requires_grad_() for c in Z]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), tokens.cuda())
    assert y.log_probs.coeffs[1][3].isnan() and y.entropy.coeffs[1][3].isfinite()
    grads = torch.autograd.grad((*y.log_probs.coeffs, *y.entropy.coeffs), leaves, [torch.ones(4, device="cuda")] * 6)
    keep = torch.arange(classes) % 2 == 1
    keep[4] = True
    z64 = [c[:1, keep].double().requires_grad_() for c in Z]
    want = series64.log_probs(z64, torch.tensor([int(keep[:4].sum())]))
    ref = torch.autograd.grad(want[0] + want[1], z64, [torch.ones(1).double()] * 6)
    for g, r in zip(grads, ref):
        g = g.cpu()
        assert not g[0, ~keep].any() and not g[1].any() and g[3].isnan().all() and g[2].isfinite().all()
        assert (g[0, keep].double() - r[0]).abs().max() <= 2 * _bound(2, classes, dtype, r)


def test_entropy_gradient_beside_a_token_that_is_no_class():
    # the token has no part in the entropy: its gradient is finite, the log probability's is not
    Z = _series((2, 300), 1, 28, torch.float64)
    tokens = torch.tensor([300, 5])
    z64 = [c.clone().requires_grad_() for c in Z]
    ref = torch.autograd.grad(series64.log_probs(z64, torch.tensor([0, 5]))[1], z64, [torch.ones(2).double()] * 2)
    leaves = [c.cuda().requires_grad_() for c in Z]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), tokens.cuda())
    ones = [torch.ones(2, dtype=torch.float64, device="cuda")] * 2
    _check_gradient(torch.autograd.grad(y.entropy.coeffs, leaves, ones, retain_graph=True), list(ref), 300, torch.float64)
    assert torch.autograd.grad(y.log_probs.coeffs, leaves, ones)[0][0].isnan().all()


def test_outputs_changed_in_place_before_the_gradient():
    Z, tokens = _series((4, 200), 1, 29, torch.float64), _tokens(4, 200, 30)
    results = []
    for change in (False, True):
        leaves = [c.cuda().requires_grad_() for c in Z]
        with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
            y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), tokens.cuda(), top=2)
        if change:
            for c in (*y.log_probs.coeffs, *y.entropy.coeffs):
                c.data.zero_()
        results.append(torch.autograd.grad([*y.log_probs.coeffs, *y.entropy.coeffs], leaves, [torch.ones(4, dtype=torch.float64, device="cuda")] * 4))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_gradient_against_differences():
    Z, tokens = _series((3, 40), 2, 17, torch.float64, 1.0), torch.tensor([3, 39, 0])
    cots = [_series((3,), 2, 18, torch.float64, 1.0), _series((3,), 2, 19, torch.float64, 1.0), _series((3, 2), 2, 20, torch.float64, 1.0)]

    def value(Z):
        y = _run(Z, tokens, top=2, softcap=6.0)
        return sum((a.cpu() * b).sum().item() for s, c in zip((y.log_probs, y.entropy, y.top_log_probs), cots)
                   for a, b in zip(s.coeffs, c))

    leaves = [c.cuda().requires_grad_() for c in Z]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), tokens.cuda(), top=2, softcap=6.0)
    outs = [c for s in (y.log_probs, y.entropy, y.top_log_probs) for c in s.coeffs]
    grads = torch.autograd.grad(outs, leaves, [c.cuda() for s in cots for c in s])
    h = 1e-5   # central differences: error h^2 times third derivatives of order ten, and rounding 2^-53 10 / h
    for i in range(3):
        d = torch.randn(Z[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        moved = lambda s: value([c + s * d if j == i else c for j, c in enumerate(Z)])   # noqa: E731
        slope, got = (moved(h) - moved(-h)) / (2 * h), (grads[i].cpu() * d).sum().item()
        assert abs(slope - got) <= 1e-6 * max(1.0, abs(got))


def test_leading_dimensions_strides_and_orders():
    dtype = torch.float32
    Z, tokens = _series((2, 3, 77), 2, 21, dtype), _tokens(6, 77, 22).view(2, 3)
    want = series64.log_probs([c.double().flatten(0, 1) for c in Z], tokens.flatten(), top=3)
    shapes = {"three": lambda c: c, "padded": lambda c: torch.nn.functional.pad(c, (2, 5))[..., 2:-5],
              "transposed": lambda c: c.transpose(1, 2).contiguous().transpose(1, 2), "offset": lambda c: torch.cat(
                  (c.new_zeros(1), c.flatten()))[1:].view(c.shape)}
    for name, shape in shapes.items():
        z = PolyTensor._wrap(tuple(shape(c.cuda()) for c in Z))
        with torch.no_grad(), PolyTensor.plain_range():
            y = PolyTensor.token_log_probs(z, tokens.cuda(), top=3)
        assert y.log_probs.shape == (2, 3) and y.top_tokens.shape == (2, 3, 3) and y.top_log_probs.shape == (2, 3, 3)
        for k in range(3):
            _check([y.log_probs.coeffs[k].flatten()], [want[0][k]], 77, dtype, name)
            _check([y.top_log_probs.coeffs[k].flatten(0, 1)], [want[3][k]], 77, dtype, name)
    with torch.no_grad(), PolyTensor.plain_range():   # one row without leading dimensions; rows behind a gap
        one = PolyTensor.token_log_probs(_poly([c[0, 0] for c in Z]), tokens[0, 0].cuda())
        wide = torch.randn(5, 200, device="cuda")
        part = PolyTensor.token_log_probs(PolyTensor._wrap((wide[:, 3:150],)), torch.arange(5, device="cuda"))
    assert one.log_probs.shape == () and abs(one.log_probs.value.item() - want[0][0][0].item()) <= _bound(2, 77, dtype, want[0][0])
    column = torch.randn(60, 1, device="cuda")   # one row whose stride is below its length
    with torch.no_grad(), PolyTensor.plain_range():
        row = PolyTensor.token_log_probs(PolyTensor._wrap((column.t(),)), torch.tensor([7], device="cuda"))
    _check(row.log_probs.coeffs, series64.log_probs([column.t().cpu().double()], torch.tensor([7]))[0], 60, dtype, "row")
    ref = series64.log_probs([wide[:, 3:150].cpu().double()], torch.arange(5))
    _check(part.log_probs.coeffs, ref[0], 147, dtype, "gap")
    # gradients through leading dimensions
    z = PolyTensor(tuple(c.cuda() for c in Z), requires_grad=True)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        PolyTensor.token_log_probs(z, tokens.cuda()).log_probs.sum().backward()
        assert z.grad.shape == z.shape and all(c.isfinite().all() for c in z.grad.coeffs)


def test_agreement_with_cross_entropy():
    Z, tokens = _series((64, 1000), 3, 23, torch.float32), _tokens(64, 1000, 24)
    y = _run(Z, tokens)
    with torch.no_grad(), PolyTensor.plain_range():
        loss = PolyTensor.cross_entropy(_poly(Z), tokens.cuda(), reduction="none")
    for a, b in zip(y.log_probs.coeffs, loss.coeffs):
        assert (a + b).abs().max() <= 2 * _bound(3, 1000, torch.float32, a)


def test_complex_directions():
    base, real, imag = _series((3, 50), 2, 25, torch.float64)
    x = [base, torch.complex(real, imag), torch.complex(imag, real)]
    tokens = torch.tensor([4, -100, 49])
    got = _run(x, tokens, top=3)
    z = [c.to(torch.complex128) for c in x]
    m = base.amax(1, keepdim=True)
    e = series64.exp([z[0] - m] + z[1:])
    lse = series64.log([c.sum(1, keepdim=True) for c in e])
    logp = [a - b for a, b in zip(z, [lse[0] + m] + lse[1:])]
    ent = [-c.sum(1) for c in series64.mul(series64.exp(logp), logp)]
    ids = base.topk(3, dim=1).indices
    for row in (0, 2):
        assert torch.equal(got.top_tokens[row].cpu(), ids[row])
        for k in range(3):
            for a, b in ((got.log_probs, logp[k][row, tokens[row]]), (got.entropy, ent[k][row]), (got.top_log_probs, logp[k][row, ids[row]])):
                a = a.coeffs[k][row].cpu()
                assert (a - (b.real if k == 0 else b)).abs().max() <= 1e-11
    assert not got.log_probs.coeffs[2][1].abs().any() and (got.top_tokens[1] == -1).all()


def test_captured_step_and_two_graphs():
    # two captured graphs and eager work in between, on logits that change from replay to replay; few rows,
    # so that the rows are cut into pieces that meet in the workspace
    rows, classes, top = 4, 30000, 8
    steps = []
    for seed in (31, 32):
        leaves = [c.cuda().requires_grad_() for c in _series((rows, classes), 2, seed, torch.float32)]
        tokens = _tokens(rows, classes, seed).cuda()
        ones = [torch.ones(rows, device="cuda") for _ in range(6)]

        def step(leaves=leaves, tokens=tokens, ones=ones):
            with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
                y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), tokens, top=top)
            grads = torch.autograd.grad((*y.log_probs.coeffs, *y.entropy.coeffs), leaves, ones)
            return [c.detach() for s in (y.log_probs, y.entropy, y.top_log_probs) for c in s.coeffs] + [y.top_tokens, *grads]

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        steps.append((graph, out, step, leaves))
    for i in range(3):
        for graph, _, _, leaves in steps:
            leaves[0].data.copy_(torch.roll(leaves[0].data, 1, 1))
            graph.replay()
        torch.cuda.synchronize()
        for _, out, step, _ in steps:
            for a, b in zip(out, step()):
                assert torch.equal(a, b), i


def test_more_elements_than_32_bits_count():
    rows, classes = 70001, 32000   # 2.24e9 logits
    z = torch.empty(rows, classes, dtype=torch.bfloat16, device="cuda").normal_()
    tokens = torch.randint(0, classes, (rows,), device="cuda")
    with torch.no_grad(), PolyTensor.plain_range():
        y = PolyTensor.token_log_probs(PolyTensor((z,)), tokens, top=3)
    last = slice(rows - 4, rows)
    want = series64.log_probs([z[last].cpu().double()], tokens[last].cpu(), top=3)
    _check([y.log_probs.value[last]], want[0], classes, torch.bfloat16, "log_probs")
    assert torch.equal(y.top_tokens[last].cpu(), want[2])
    ones = [torch.ones(rows, device="cuda")]
    raw = torch.ops.polytensors_amd.token_log_probs_series([z], tokens, -100, 0.0, 0)
    dz = torch.ops.polytensors_amd.token_log_probs_series_backward([z], tokens, -100, 0.0, raw[4], raw[1], None, ones, [], [])[0]
    z64 = z[last].cpu().double().requires_grad_()
    (ref,) = torch.autograd.grad(series64.log_probs([z64], tokens[last].cpu())[0][0].sum(), z64)
    _check_gradient([dz[last]], [ref], classes, torch.bfloat16)


def test_empty_and_refused_calls():
    Z, tokens = _series((4, 10), 1, 26, torch.float32), _tokens(4, 10, 27)
    z, t = _poly(Z), tokens.cuda()
    bad = [((Z[0].cuda(), t), {}, "PolyTensor"), ((z, tokens), {}, "tokens"), ((z, t.int()), {}, "tokens"), ((z, t[:3]), {}, "tokens"),
           ((z, t), dict(top=33), "top"), ((z, t), dict(top=11), "top"), ((z, t), dict(top=-1), "top"), ((z, t), dict(top=True), "top"),
           ((z, t), dict(top=1.0), "top"), ((z, t), dict(softcap=0.0), "softcap"), ((z, t), dict(softcap=-1.0), "softcap"),
           ((z, t), dict(softcap=INF), "softcap"), ((z, t), dict(ignore_index=0.5), "ignore_index"),
           ((PolyTensor((Z[0].cuda(),), degree=9), t), {}, "degree 9"),
           ((PolyTensor((torch.empty(4, 0, device="cuda"),)), t), {}, "class")]
    with torch.no_grad(), PolyTensor.plain_range():
        for args, kwargs, needle in bad:
            with pytest.raises(NotImplementedError, match=needle):
                PolyTensor.token_log_probs(*args, **kwargs)
        y = PolyTensor.token_log_probs(PolyTensor((torch.empty(0, 10, device="cuda"),), degree=2),
                                       torch.empty(0, dtype=torch.int64, device="cuda"), top=2)
        assert y.log_probs.shape == (0,) and y.top_tokens.shape == (0, 2) and y.top_log_probs.degree == 2
    with pytest.raises(NotImplementedError, match="plain_range"):
        PolyTensor.token_log_probs(z, t)
    leaves = [c.cuda().requires_grad_() for c in Z]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y = PolyTensor.token_log_probs(PolyTensor(tuple(leaves)), t)
        with pytest.raises(NotImplementedError, match="second-order"):
            torch.autograd.grad(y.log_probs.value.sum(), leaves[0], create_graph=True)
