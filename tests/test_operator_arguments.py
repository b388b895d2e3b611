"""Argument errors of the dropout, norm-and-rotation and log-probability entry points (CPU: no launch), and
the shapes of their operators without a device."""

import ctypes

import pytest
import torch

from polytensors_amd import _lib, _ops


def _vpp(n):
    return (ctypes.c_void_p * n)(*([1 << 20] * n))


def _operand(**kwargs):
    op = _lib.NormRopeOperand()
    keep = dict(x=_vpp(2), stride_b=64, stride_l=64, stride_h=8, heads=8, weight=None, weight_orders=0, y=_vpp(2), grad=_vpp(2),
                dx=_vpp(2), dweight=None, dweight_orders=0)
    keep.update(kwargs)
    for name, value in keep.items():
        if value is not None:
            setattr(op, name, ctypes.cast(value, ctypes.POINTER(ctypes.c_void_p)) if isinstance(value, ctypes.Array) else value)
    op._keep = keep
    return op


def _rope(direction="fwd", op=None, dtype=0, degree=1, n=1, batch=1, length=1, dim=8, rotary=8, rows=4, tables=1 << 20, stride=0,
          eps=1e-5, workspace=None):
    lib = _lib.load()
    op = _operand() if op is None else op
    args = [dtype, degree, n, ctypes.addressof(op), batch, length, dim, rotary, 0, tables, tables, rows, None, stride, eps]
    if direction == "bwd":
        args.append(workspace)
    status = getattr(lib, f"pt_norm_rope_series_{direction}")(*args, None)
    return status, lib.pt_last_error().decode()


@pytest.mark.parametrize("kwargs,status,needle", [
    (dict(degree=9), 2, "degree"), (dict(dtype=9), 2, "dtype"), (dict(n=3), 1, "operands"), (dict(n=0), 1, "operands"),
    (dict(dim=257), 2, "head_dim"), (dict(dim=0), 2, "head_dim"), (dict(rotary=7), 1, "rotary"), (dict(rotary=10), 1, "rotary"),
    (dict(tables=None), 1, "tables"), (dict(stride=-1), 1, "stride"), (dict(eps=-1.0), 1, "eps"), (dict(eps=float("nan")), 1, "eps"),
    (dict(batch=-1), 1, "batch"), (dict(batch=1 << 20, length=1 << 20), 2, "2^31"),
    (dict(op=_operand(heads=0)), 1, "heads"), (dict(op=_operand(stride_h=-8)), 1, "stride"),
    (dict(op=_operand(weight_orders=1)), 1, "weight_orders"), (dict(op=_operand(weight_orders=3, weight=_vpp(3))), 1, "weight_orders"),
    (dict(direction="bwd", op=_operand(dweight_orders=1, dweight=_vpp(1))), 1, "workspace"),
    (dict(direction="bwd", op=_operand(dweight_orders=3, dweight=_vpp(3))), 1, "dweight_orders"),
])
def test_norm_rope_errors(kwargs, status, needle):
    got, message = _rope(**kwargs)
    assert got == status and needle in message


def test_norm_rope_of_nothing_and_workspace():
    assert _rope(batch=0) == (0, "") and _rope(direction="bwd", length=0) == (0, "")
    size = _lib.load().pt_norm_rope_series_bwd_workspace_size
    assert size(0, 2, 100, 64) == 100 * 3 * 64 * 4 and size(1, 2, 1 << 20, 64) == 1024 * 3 * 64 * 8
    assert size(0, 9, 100, 64) == 0 and size(0, 2, 0, 64) == 0


@pytest.mark.parametrize("args,status,needle", [
    ((0, 0, _vpp(1), _vpp(1), 4, 0.5, 1 << 20, None), 2, "orders"), ((0, 18, _vpp(18), _vpp(18), 4, 0.5, 1 << 20, None), 2, "orders"),
    ((4, 1, _vpp(1), _vpp(1), 4, 0.5, 1 << 20, None), 2, "dtype"), ((0, 1, _vpp(1), _vpp(1), 4, 1.5, 1 << 20, None), 1, "p must"),
    ((0, 1, _vpp(1), _vpp(1), 4, float("nan"), 1 << 20, None), 1, "p must"), ((0, 1, _vpp(1), _vpp(1), -1, 0.5, 1 << 20, None), 1, "numel"),
    ((0, 1, _vpp(1), _vpp(1), 4, 0.5, None, None), 1, "seed"), ((0, 1, None, _vpp(1), 4, 0.5, 1 << 20, None), 1, "required"),
    ((0, 1, _vpp(1), _vpp(1), 0, 0.5, 1 << 20, None), 0, ""),
])
def test_dropout_errors(args, status, needle):
    lib = _lib.load()
    assert lib.pt_dropout_series(*args) == status and needle in lib.pt_last_error().decode()


def _log_probs(dtype=0, degree=1, z=True, rows=4, classes=10, stride=10, tokens=1 << 20, softcap=0.0, top=0, outs=True, ids=1 << 20,
               tops=True, workspace=None):
    p = lambda on: _vpp(2) if on else None   # noqa: E731
    lib = _lib.load()
    status = lib.pt_token_log_probs_series_fwd(dtype, degree, p(z), rows, classes, stride, tokens, -100, softcap, top, p(outs),
                                               p(True), ids, p(tops), p(True), workspace, None)
    return status, lib.pt_last_error().decode()


@pytest.mark.parametrize("kwargs,status,needle", [
    (dict(degree=9), 2, "degree"), (dict(dtype=7), 2, "dtype"), (dict(z=False), 1, "logits"), (dict(classes=0), 1, "classes"),
    (dict(stride=9), 1, "row_stride"), (dict(classes=1 << 31, stride=1 << 31), 2, "classes"), (dict(rows=1 << 31), 2, "rows"),
    (dict(tokens=None), 1, "tokens"), (dict(softcap=-1.0), 1, "softcap"), (dict(softcap=float("nan")), 1, "softcap"),
    (dict(top=33, classes=100, stride=100), 1, "top"), (dict(top=11), 1, "top"), (dict(top=-1), 1, "top"),
    (dict(outs=False), 1, "log_probs"), (dict(top=2, ids=None), 1, "top_tokens"), (dict(top=2, tops=False), 1, "top_log_probs"),
    (dict(classes=1 << 17, stride=1 << 17), 1, "workspace"), (dict(rows=0), 0, ""),
])
def test_log_probs_errors(kwargs, status, needle):
    got, message = _log_probs(**kwargs)
    assert got == status and needle in message


def test_log_probs_workspace():
    size = _lib.load().pt_token_log_probs_series_workspace_size
    assert size(0, 2, 4096, 32000, 5) == 0 and size(0, 2, 4, 500, 5) == 0     # rows enough, or too short to cut
    few = size(0, 2, 4, 1 << 17, 5)                                           # 64 pieces a row
    assert few == 4 * 64 * (4 * (5 + 9) + 4 * 5)
    assert size(0, 9, 4, 1 << 17, 5) == 0 and size(0, 2, 4, 1 << 17, 33) == 0


def test_log_probs_backward_errors():
    lib = _lib.load()
    call = lambda *a: lib.pt_token_log_probs_series_bwd(0, 1, _vpp(2), 4, 10, 10, 1 << 20, -100, 0.0, *a, None)   # noqa: E731
    assert call(0, None, _vpp(2), _vpp(2), None, None, _vpp(2), _vpp(2)) == 1 and "top_tokens" in lib.pt_last_error().decode()
    assert call(0, None, None, _vpp(2), None, None, None, _vpp(2)) == 1 and "lse" in lib.pt_last_error().decode()
    assert call(0, None, _vpp(2), _vpp(2), None, None, None, None) == 1 and "dz" in lib.pt_last_error().decode()


def test_shapes_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    if not _ops.NATIVE:
        pytest.skip("libpolytaylor_torch.so is not built")
    with FakeTensorMode():
        x = [torch.empty(2, 3, 4, 8, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
        k = [c[:, :, :2] for c in x]
        tables = torch.empty(5, 4, device="cuda")
        q_out, k_out = _ops.norm_rope_series(x, k, tables, tables, None, [], [], 1e-5, False)
        assert q_out.shape == (3, 2, 4, 3, 8) and k_out.shape == (3, 2, 2, 3, 8)
        assert len(_ops.norm_rope_series_orders(x, k, tables, tables, None, [], [], 1e-5, False)) == 6
        z = [torch.empty(6, 50, device="cuda", dtype=torch.float16) for _ in range(2)]
        out = _ops.token_log_probs_series(z, torch.empty(6, device="cuda", dtype=torch.int64), -100, 0.0, 4)
        assert [tuple(t.shape) for t in out] == [(2, 6), (2, 6), (6, 4), (2, 6, 4), (2, 6)] and out[0].dtype == torch.float32
        assert _ops.dropout_series(z, torch.empty(1, device="cuda", dtype=torch.int64), 0.5).shape == (2, 6, 50)
