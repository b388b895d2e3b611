"""The float64 test helper against independent values (CPU): nested forward-mode derivatives of torch's own
operations, and published outputs of the generator."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from tests import series64
from tests.jets import rel_err, taylor


def _series(shape, degree, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g, dtype=torch.float64) * 0.5 ** k for k in range(degree + 1)]


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_is_the_series_of_the_plain_operation(interleaved):
    degree = 3
    x, w = _series((2, 3, 2, 6), degree, 1), _series((6,), degree, 2)
    angle = torch.arange(8, dtype=torch.float64)[:, None] * torch.tensor([1.0, 0.3], dtype=torch.float64)
    positions = torch.tensor([[0, 5, 7], [2, 2, 1]])

    def plain(x, w):
        y = F.rms_norm(x, (6,), w, 1e-5)
        first = y[..., 0:4:2] if interleaved else y[..., 0:2]
        second = y[..., 1:4:2] if interleaved else y[..., 2:4]
        turned = torch.complex(first, second) * torch.polar(torch.ones(()).double(), angle[positions])[:, :, None]
        pair = (turned.real, turned.imag)
        turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
        return torch.cat((turned, y[..., 4:]), -1).transpose(1, 2)

    got = series64.norm_rope(x, w, angle.cos(), angle.sin(), positions, 1e-5, interleaved)
    for a, b in zip(got, taylor(plain, [x, w], degree)):
        assert rel_err(a, b) < 1e-13


@pytest.mark.parametrize("softcap", [None, 3.0])
def test_log_probs_are_the_series_of_the_plain_operation(softcap):
    degree = 3
    z = _series((4, 9), degree, 3)
    tokens = torch.tensor([0, 8, -100, 3])
    cap = (lambda z: z) if softcap is None else (lambda z: softcap * torch.tanh(z / softcap))
    keep = (tokens != -100).double()
    got = series64.log_probs(z, tokens, top=3, softcap=softcap)
    want = taylor(lambda z: torch.log_softmax(cap(z), 1)[range(4), tokens.clamp_min(0)] * keep, [z], degree)
    ent = taylor(lambda z: -(torch.softmax(cap(z), 1) * torch.log_softmax(cap(z), 1)).sum(1) * keep, [z], degree)
    ids = z[0].topk(3, dim=1).indices
    tops = taylor(lambda z: torch.log_softmax(cap(z), 1).gather(1, ids) * keep[:, None], [z], degree)
    assert torch.equal(got[2], torch.where(tokens[:, None] == -100, -1, ids))
    for k in range(degree + 1):
        assert rel_err(got[0][k], want[k]) < 1e-12
        assert rel_err(got[1][k], ent[k]) < 1e-12
        assert rel_err(got[3][k], tops[k]) < 1e-12


def test_generator_published_outputs():
    # the generator's authors' known answers for Philox4x32-10: counter and key all zero; and word order
    assert [hex(v) for v in series64.philox(0, 4, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    whole = series64.philox(0, 64, 123)
    assert np.array_equal(series64.philox(5, 20, 123), whole[5:25])
    assert np.array_equal(series64.philox(4, 4, -1), series64.philox(4, 4, 2 ** 64 - 1))
