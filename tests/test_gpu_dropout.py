"""Dropout of a series on the GPU: the mask against the generator's plain form, values exactly.

y = x / (1 - p) rounded once where the mask keeps, 0 elsewhere: the product in the arithmetic type is the
plain form's, so kernel and plain form agree in every bit and no tolerance is needed.
"""

import pytest
import torch
import torch.nn.functional as F

from polytensors_amd import PolyTensor
from tests import series64

pytestmark = pytest.mark.gpu

DTYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def _series(shape, degree, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(shape, generator=g, dtype=torch.float64) * 0.5 ** k).to(dtype) for k in range(degree + 1)]


def _want(c, seed, p):
    acc = torch.float64 if c.dtype == torch.float64 else torch.float32
    kept = series64.keep(0, c.numel(), seed, p).view(c.shape)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=acc)
    return torch.where(kept & (p < 1), c.to(acc) * scale, 0.0).to(c.dtype)


def _seed(value):
    return torch.tensor([value], device="cuda")


@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7,), (8,), (255,), (1000, 3), (5, 7, 9), (33, 1024)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_is_the_generators_mask(shape, dtype):
    for degree, seed, p in ((0, 0, 0.5), (2, -1, 0.1), (3, 2 ** 62 + 12345, 0.9)):
        X = _series(shape, degree, 1, dtype)
        x = PolyTensor(tuple(c.cuda() for c in X))
        with torch.no_grad(), PolyTensor.plain_range():
            y = PolyTensor.dropout(x, p, seed=_seed(seed))
            again = PolyTensor.dropout(x, p, seed=seed)
        assert y.degree == degree and y.dtype == dtype
        for k in range(degree + 1):
            assert torch.equal(y.coeffs[k].cpu(), _want(X[k], seed, p)), (degree, k)
            assert torch.equal(y.coeffs[k], again.coeffs[k])


@pytest.mark.parametrize("degree", [1, 4, 5, 6, 7, 8, 9, 16])
def test_every_degree(degree):
    X = _series((13, 21), degree, 2, torch.float32)
    with torch.no_grad(), PolyTensor.plain_range():
        y = PolyTensor.dropout(PolyTensor(tuple(c.cuda() for c in X)), 0.3, seed=7)
    for k in range(degree + 1):
        assert torch.equal(y.coeffs[k].cpu(), _want(X[k], 7, 0.3))


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_at_any_element_and_in_any_order(dtype):
    X = _series((9, 41), 2, 3, dtype)
    views = [lambda c: c[:, 1:], lambda c: c.t(), lambda c: c.flatten()[5:], lambda c: c[::2, ::3],
             lambda c: c[3:4].expand(6, 41)]
    for view in views:
        with torch.no_grad(), PolyTensor.plain_range():
            x = PolyTensor(tuple(c.cuda() for c in X))
            x = PolyTensor._wrap(tuple(view(c) for c in x.coeffs))
            y = PolyTensor.dropout(x, 0.4, seed=11)
        for k in range(3):   # the mask goes by the view's own row-major index
            assert torch.equal(y.coeffs[k].cpu(), _want(view(X[k]).contiguous(), 11, 0.4))


def test_the_ends_of_p_and_numbers_that_are_none():
    x = torch.tensor([1.0, float("nan"), float("inf"), -2.0, 5.0], device="cuda")
    X = PolyTensor((x, x.clone()))
    with torch.no_grad(), PolyTensor.plain_range():
        none = PolyTensor.dropout(X, 0.0, seed=3)
        every = PolyTensor.dropout(X, 1.0, seed=3)
        some = PolyTensor.dropout(X, 0.5, seed=3)
    assert torch.equal(none.value.nan_to_num(9.0), x.nan_to_num(9.0)) and not every.value.any()
    kept = series64.keep(0, 5, 3, 0.5)
    assert torch.equal(some.value.cpu() == 0, ~kept)   # a dropped NaN is zero
    largest = 1.0 - 2.0 ** -53
    with torch.no_grad(), PolyTensor.plain_range():
        y = PolyTensor.dropout(PolyTensor((torch.ones(4096, device="cuda"),)), largest, seed=3)
    assert torch.equal(y.value.cpu() != 0, series64.keep(0, 4096, 3, largest))


def test_functional_and_module():
    x = PolyTensor(tuple(c.cuda() for c in _series((64, 64), 2, 4, torch.float32)))
    with torch.no_grad(), PolyTensor.plain_range():
        assert F.dropout(x, 0.5, training=False) is x and F.dropout(x, 0.0) is x
        assert torch.dropout(x, 0.5, False) is x
        torch.manual_seed(5)
        a = F.dropout(x, 0.25)
        b = F.dropout(x, 0.25)
        torch.manual_seed(5)
        c = torch.nn.Dropout(0.25)(x)
        assert torch.equal(a.value, c.value) and not torch.equal(a.value, b.value)
        kept = a.value != 0
        assert torch.equal(kept, a.coeffs[2] != 0) and torch.equal(a.coeffs[1], x.coeffs[1] * kept * (1.0 / 0.75))
        # 4096 elements kept with 3/4: six standard deviations of the rate are 0.041
        assert abs(kept.double().mean().item() - 0.75) < 0.041
        for bad in (-0.1, 1.5):
            with pytest.raises(ValueError):
                F.dropout(x, bad)
        with pytest.raises(NotImplementedError, match="inplace"):
            F.dropout(x, 0.5, inplace=True)


def test_wrapper_gradient_is_the_same_mask():
    X, C = _series((31, 17), 3, 5, torch.float32), _series((31, 17), 3, 6, torch.float32)
    x = PolyTensor(tuple(c.cuda() for c in X), requires_grad=True)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        y = PolyTensor.dropout(x, 0.2, seed=9)
        y.backward(PolyTensor(tuple(c.cuda() for c in C)))
        for k in range(4):
            assert torch.equal(x.grad.coeffs[k].cpu(), _want(C[k], 9, 0.2))


def test_coefficient_gradients_and_their_derivative():
    X, C = _series((12, 5), 2, 7, torch.float64), _series((12, 5), 2, 8, torch.float64)
    leaves = [c.cuda().requires_grad_() for c in X]
    cots = [c.cuda().requires_grad_() for c in C]
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y = PolyTensor.dropout(PolyTensor(tuple(leaves)), 0.5, seed=10)
        grads = torch.autograd.grad(y.coeffs, leaves, cots, create_graph=True)
        second = torch.autograd.grad([(g * g).sum() for g in grads], cots)
    for k in range(3):
        want = _want(C[k], 10, 0.5)
        assert torch.equal(grads[k].detach().cpu(), want)
        assert torch.equal(second[k].cpu(), _want(2 * want, 10, 0.5))


def test_wrapper_gradient_differentiates_again():
    X, C = _series((6, 7), 1, 30, torch.float64), _series((6, 7), 1, 31, torch.float64)
    x = PolyTensor(tuple(c.cuda() for c in X), requires_grad=True)
    c = PolyTensor(tuple(t.cuda() for t in C), requires_grad=True)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        y = PolyTensor.dropout(x, 0.5, seed=32)
        (dx,) = torch.autograd.grad((y,), (x,), (c,), create_graph=True)
        (dc,) = torch.autograd.grad((dx,), (c,), (PolyTensor(tuple(t.cuda() for t in X)),))
        for k in range(2):
            assert torch.equal(dx.coeffs[k].detach().cpu(), _want(C[k], 32, 0.5))
            assert torch.equal(dc.coeffs[k].cpu(), _want(X[k], 32, 0.5))


def test_a_seed_changed_before_the_gradient_is_an_error():
    x = [torch.ones(8, device="cuda", requires_grad=True)]
    seed = _seed(1)
    with PolyTensor.plain_range(), PolyTensor.coefficient_autograd():
        y = PolyTensor.dropout(PolyTensor(tuple(x)), 0.5, seed=seed)
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.coeffs[0].sum(), x[0])


@pytest.mark.parametrize("recorded", [False, True])
def test_complex_directions(recorded):
    X = _series((9, 8), 2, 12, torch.float32)
    planes = [X[0]] + [torch.complex(c, c.flip(0)) for c in X[1:]]
    x = PolyTensor(tuple(c.cuda() for c in planes), requires_grad=recorded)
    with torch.set_grad_enabled(recorded), PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        y = PolyTensor.dropout(x, 0.3, seed=13)
        for k in range(3):
            got, c = y.coeffs[k].detach().cpu(), planes[k]
            if k == 0:
                assert torch.equal(got, _want(c, 13, 0.3))
            else:
                assert torch.equal(got.real, _want(c.real.contiguous(), 13, 0.3))
                assert torch.equal(got.imag, _want(c.imag.contiguous(), 13, 0.3))
        if recorded:
            y.backward(PolyTensor(tuple(c.cuda() for c in planes)))
            assert torch.equal(x.grad.coeffs[2].cpu(), y.coeffs[2].detach().cpu())


def test_captured_graph_reads_the_seed_at_each_replay():
    x = PolyTensor(tuple(c.cuda() for c in _series((100, 33), 2, 14, torch.bfloat16)))
    seed = _seed(1)
    with torch.no_grad(), PolyTensor.plain_range():
        PolyTensor.dropout(x, 0.5, seed=seed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = PolyTensor.dropout(x, 0.5, seed=seed)
        for value in (5, 6, 5):
            seed.fill_(value)
            graph.replay()
            torch.cuda.synchronize()
            eager = PolyTensor.dropout(x, 0.5, seed=value)
            assert all(torch.equal(a, b) for a, b in zip(y.coeffs, eager.coeffs))


def test_functional_in_a_captured_graph_draws_a_new_mask():
    x = PolyTensor(tuple(c.cuda() for c in _series((64, 64), 1, 15, torch.float32)))
    with torch.no_grad(), PolyTensor.plain_range():
        F.dropout(x, 0.5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = F.dropout(x, 0.5)
        masks = []
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            masks.append(y.value != 0)
            assert torch.equal(y.coeffs[1], x.coeffs[1] * masks[-1] * 2.0)
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])


def test_another_stream():
    X = _series((500, 77), 1, 16, torch.float32)
    stream = torch.cuda.Stream()
    x = PolyTensor(tuple(c.cuda() for c in X))
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.no_grad(), PolyTensor.plain_range():
        y = PolyTensor.dropout(x, 0.1, seed=17)
    stream.synchronize()
    assert torch.equal(y.value.cpu(), _want(X[0], 17, 0.1))


def test_more_elements_than_32_bits_count():
    n = 2 ** 32 + 37
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad(), PolyTensor.plain_range():
        y = PolyTensor.dropout(PolyTensor((x,)), 0.5, seed=18).value
    for first in (0, 2 ** 31 - 50, 2 ** 32 - 65, n - 100):
        assert torch.equal(y[first:first + 100].cpu() != 0, series64.keep(first, 100, 18, 0.5)), first


def test_empty_and_refused_calls():
    with torch.no_grad(), PolyTensor.plain_range():
        empty = PolyTensor.dropout(PolyTensor((torch.empty(0, 3, device="cuda"),), degree=1), 0.5, seed=1)
        assert empty.shape == (0, 3) and empty.degree == 1
        x = PolyTensor((torch.ones(4, device="cuda"), torch.ones(4, device="cuda")))
        for p in (-0.1, 1.1, float("nan"), True, "0.5"):
            with pytest.raises(ValueError):
                PolyTensor.dropout(x, p, seed=1)
        for seed in (True, 2 ** 63, 1.5):
            with pytest.raises(ValueError):
                PolyTensor.dropout(x, 0.5, seed=seed)
        for seed in (torch.tensor([1]), torch.tensor([1.0], device="cuda"), torch.tensor([1, 2], device="cuda")):
            with pytest.raises(NotImplementedError, match="seed"):
                PolyTensor.dropout(x, 0.5, seed=seed)
        with pytest.raises(NotImplementedError, match="PolyTensor"):
            PolyTensor.dropout(torch.ones(4, device="cuda"), 0.5)
        with pytest.raises(NotImplementedError, match="degree 17"):
            PolyTensor.dropout(PolyTensor((torch.ones(4, device="cuda"),), degree=17), 0.5)
    with pytest.raises(NotImplementedError, match="plain_range"):
        PolyTensor.dropout(x, 0.5)
