"""Norms, gated activations, adapters and 8-bit activations without a device: what the C ABI refuses before it touches
one, workspace sizes, the rule of 8 bits, and what the Python calls refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_offload import _native, adapters, gated, norms
from moss_offload.kept8 import Kept8, checkpoint_kept8, keep8

import kept8_model

P = 1 << 20  # an address that nothing reads


def _refused(status: int) -> str:
    assert status == _native.MO_E_INVALID
    return _native.load().mo_last_error().decode()


def _norm(**fields):
    call = _native.MoNormCall()
    for name in ("x", "out", "grad", "stats", "weight", "weight_grad"):
        setattr(call, name, P)
    call.rows, call.dim, call.x_stride, call.grad_stride, call.dtype, call.weight_dtype, call.scale_dtype = 10, 64, 64, 64, 1, 2, 1
    for name, value in fields.items():
        setattr(call, name, value)
    return call


@pytest.mark.parametrize("fields", [
    {"x": 0}, {"out": 0}, {"x": P + 1}, {"out": P + 1}, {"dtype": 3}, {"weight_dtype": 3}, {"scale_dtype": 3}, {"rows": 0},
    {"rows": 1 << 31}, {"dim": 0}, {"dim": 16385}, {"x_stride": 63}, {"weight": P + 2}, {"scale": P}, {"scale": P, "samples": 3},
    {"samples": 2}, {"scale": P, "samples": 2, "cu": P + 4}, {"cu": P}, {"scale": P + 1, "samples": 2}, {"stats": P + 2},
    {"scale": P, "samples": 1 << 16, "cu": P}])
def test_the_norms_refuse(fields) -> None:
    lib = _native.load()
    call = _norm(**fields)
    _refused(lib.mo_norm_forward(ctypes.byref(call), 0))
    _refused(lib.mo_norm_backward(ctypes.byref(call), P, 1 << 40, 0))
    assert lib.mo_norm_workspace_bytes(ctypes.byref(call)) == 0


@pytest.mark.parametrize("fields", [{"kept": P}, {"kept_exponents": P}, {"kept": P + 4, "kept_exponents": P}, {"x_exponents": P}])
def test_the_norms_forward_refuses(fields) -> None:
    _refused(_native.load().mo_norm_forward(ctypes.byref(_norm(**fields)), 0))


@pytest.mark.parametrize("fields", [
    {"grad": 0}, {"grad": P + 1}, {"stats": 0}, {"grad_stride": 63}, {"weight": 0}, {"bias_grad": P}, {"scale_grad": P},
    {"shift_grad": P}, {"x_exponents": P, "x": P + 4}])
def test_the_norms_backward_refuses(fields) -> None:
    _refused(_native.load().mo_norm_backward(ctypes.byref(_norm(**fields)), P, 1 << 40, 0))


def test_the_norms_workspace() -> None:
    lib = _native.load()
    call = _norm()
    needed = lib.mo_norm_workspace_bytes(ctypes.byref(call))
    assert needed and needed % 256 == 0
    for where, size in ((0, needed), (P + 8, needed), (P, needed - 1)):
        assert "workspace" in _refused(lib.mo_norm_backward(ctypes.byref(call), where, size, 0))
    assert lib.mo_norm_workspace_bytes(ctypes.byref(_norm(weight_grad=0))) == 0
    # sums for each sample beside those of the groups of rows
    more = lib.mo_norm_workspace_bytes(ctypes.byref(_norm(scale=P, samples=5)))
    assert more >= needed + (4 + 5) * 2 * 64 * 4


def _gated(**fields):
    call = _native.MoGatedCall()
    for name in ("up", "gate", "out", "out_gate", "grad"):
        setattr(call, name, P)
    call.rows, call.cols, call.dtype = 10, 64, 1
    call.up_stride = call.gate_stride = call.grad_stride = call.out_stride = 64
    for name, value in fields.items():
        setattr(call, name, value)
    return call


@pytest.mark.parametrize("fields", [
    {"up": 0}, {"gate": 0}, {"out": 0}, {"up": P + 1}, {"out": P + 1}, {"dtype": 3}, {"rows": 0}, {"rows": 1 << 31}, {"cols": 0},
    {"up_stride": 63}, {"gate_stride": 63}, {"out_stride": 63}, {"rows": 1 << 28}, {"up_exponents": P}])
def test_the_gated_activations_refuse(fields) -> None:
    lib = _native.load()
    call = _gated(**fields)
    _refused(lib.mo_gated_forward(ctypes.byref(call), 0))
    _refused(lib.mo_gated_backward(ctypes.byref(call), 0))


def test_the_gated_activations_refuse_half_of_8_bits() -> None:
    lib = _native.load()
    names = ("kept_up", "kept_gate", "kept_up_exponents", "kept_gate_exponents")
    whole = {**dict.fromkeys(names, P), "values_stride": 64, "exponents_stride": 2}
    for name in names[:2]:
        _refused(lib.mo_gated_forward(ctypes.byref(_gated(**{**whole, name: 0})), 0))
        _refused(lib.mo_gated_forward(ctypes.byref(_gated(**{**whole, name: P + 4})), 0))
    for fields in ({"kept_up_exponents": 0}, {"values_stride": 56}, {"values_stride": 68}, {"exponents_stride": 1}):
        _refused(lib.mo_gated_forward(ctypes.byref(_gated(**{**whole, **fields})), 0))
    kept = {"up_exponents": P, "gate_exponents": P, "values_stride": 64, "exponents_stride": 2}
    for fields in ({"gate_exponents": 0}, {"up": P + 4}, {"values_stride": 32}, {"grad": 0}, {"out_gate": 0}, {"grad_stride": 8}):
        _refused(lib.mo_gated_backward(ctypes.byref(_gated(**{**kept, **fields})), 0))


def test_8_bit_calls_refuse() -> None:
    lib = _native.load()
    good = {"x": P, "dtype": 1, "rows": 4, "cols": 40, "stride": 40, "values": P, "exponents": P}
    for fields in ({"x": 0}, {"values": 0}, {"exponents": 0}, {"x": P + 1}, {"values": P + 4}, {"dtype": 3}, {"rows": 0}, {"cols": 0},
                   {"rows": 1 << 31}, {"stride": 39}, {"rows": 1 << 29}, {"cols": 1 << 30}):
        c = {**good, **fields}
        _refused(lib.mo_keep_pack(c["x"], c["dtype"], c["rows"], c["cols"], c["stride"], c["values"], c["exponents"], 0))
        _refused(lib.mo_keep_restore(c["values"], c["exponents"], c["x"], c["dtype"], c["rows"], c["cols"], c["stride"], 0))


def _adapters(**fields):
    call = _native.MoAdaptersCall()
    for name in ("x", "result", "y", "a", "b", "hidden", "grad", "dx", "da", "db"):
        setattr(call, name, P)
    call.rows, call.in_features, call.out_features, call.rank, call.dtype = 12, 64, 96, 8, 1
    call.x_stride, call.result_stride, call.grad_stride, call.requests, call.adapters, call.factor = 64, 96, 96, 1, 1, 1.0
    for name, value in fields.items():
        setattr(call, name, value)
    return call


@pytest.mark.parametrize("fields", [
    {"x": 0}, {"a": 0}, {"b": 0}, {"hidden": 0}, {"a": P + 1}, {"x": P + 1}, {"hidden": P + 2}, {"dtype": 3}, {"rows": 0},
    {"rows": (1 << 31) - 65536}, {"in_features": 0}, {"out_features": (1 << 20) + 1}, {"rank": 0}, {"rank": 129}, {"requests": 0},
    {"adapters": 0}, {"adapters": 2}, {"requests": 5}, {"requests": 1 << 16, "cu": P}, {"cu": P + 4}, {"index": P + 4},
    {"scale": P + 2}, {"x_stride": 63}])
def test_the_adapters_refuse(fields) -> None:
    lib = _native.load()
    call = _adapters(**fields)
    _refused(lib.mo_adapters_forward(ctypes.byref(call), P, 1 << 40, 0))
    _refused(lib.mo_adapters_backward(ctypes.byref(call), P, 1 << 40, 0))
    assert lib.mo_adapters_workspace_bytes(ctypes.byref(call), 1) == 0


def test_the_adapters_refuse_by_direction() -> None:
    lib = _native.load()
    for fields in ({"result": 0}, {"y": 0}, {"y": P + 1}, {"result_stride": 95}, {"x_exponents": P}):
        _refused(lib.mo_adapters_forward(ctypes.byref(_adapters(**fields)), P, 1 << 40, 0))
    for fields in ({"grad": 0}, {"grad_stride": 95}, {"add": P, "add_stride": 63}, {"add": P + 1}, {"dx": 0, "da": 0, "db": 0},
                   {"x_exponents": P, "x": P + 4}):
        _refused(lib.mo_adapters_backward(ctypes.byref(_adapters(**fields)), P, 1 << 40, 0))
    needed = lib.mo_adapters_workspace_bytes(ctypes.byref(_adapters()), 1)
    assert needed % 256 == 0
    for where, size in ((0, needed), (P + 8, needed), (P, needed - 1)):
        assert "workspace" in _refused(lib.mo_adapters_backward(ctypes.byref(_adapters()), where, size, 0))


def test_tensors_off_the_device_are_refused() -> None:
    x = torch.zeros(4, 64)
    for call in (lambda: keep8(x), lambda: norms.norm_forward(x), lambda: gated.gated_forward(x),
                 lambda: adapters.adapters_forward(x, x, x[None], x[None, :, :4].expand(1, 4, 4), 1.0)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    with pytest.raises(RuntimeError, match="HIP"):
        Kept8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 2, dtype=torch.uint8), 64, torch.float32).restore()


def test_8_bit_tensors_are_checked() -> None:
    values, exponents = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    kept = Kept8(values, exponents, 50, torch.bfloat16)
    assert kept.shape == (4, 50) and kept.nbytes == 4 * 66
    for bad in ((values.float(), exponents, 50, torch.bfloat16), (values, exponents.int(), 50, torch.bfloat16),
                (values, exponents, 50, torch.float64)):
        with pytest.raises(TypeError):
            Kept8(*bad)
    for bad in ((values, exponents, 32, torch.bfloat16), (values, exponents[:3], 50, torch.bfloat16), (values, exponents, 0, torch.bfloat16),
                (values, exponents, 65, torch.bfloat16)):
        with pytest.raises(ValueError):
            Kept8(*bad)
    shifted = torch.zeros(4 * 64 + 1, dtype=torch.int8)[1:].view(4, 64)
    assert Kept8(shifted, exponents, 64, torch.bfloat16).values.data_ptr() % 8 == 0


def test_a_checkpoint_without_a_gradient_to_give_is_refused() -> None:
    with pytest.raises(RuntimeError, match="requires grad"):
        checkpoint_kept8(lambda t: t, torch.zeros(2, 3))
    with torch.no_grad():
        assert checkpoint_kept8(lambda t: t + 1, torch.zeros(2, 3)).eq(1).all()


def test_the_rule_of_8_bits() -> None:
    """The model that the kernels are held to, at values whose step is known."""

    x = torch.zeros(1, 33)
    x[0, 0], x[0, 1], x[0, 2], x[0, 32] = 127.0, 0.5, 1.5, 127.5
    values, exponents = kept8_model.keep(x)
    assert exponents.tolist() == [[127, 128]] and values[0, :3].tolist() == [127, 0, 2] and values[0, 32] == 64
    assert kept8_model.read(values, exponents, 33)[0, 32] == 128.0
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        most = torch.tensor([[torch.finfo(dtype).max]], dtype=dtype)
        back = kept8_model.read_back(most)
        assert torch.isfinite(back.to(dtype)).all() and back <= most.double() and back >= 0.98 * most.double()
    assert torch.isnan(kept8_model.read_back(torch.tensor([[1.0, float("inf")]]))).all()
    assert kept8_model.read_back(torch.tensor([[2.0**-140, 2.0**-126]])).tolist() == [[0.0, 2.0**-126]]
