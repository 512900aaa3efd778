"""Rotary positions on the CPU: the scaled bands by their formulas, and what the calls refuse."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from moss_offload import _native, rotary


def _bands(n=32):
    return (1 / 10000 ** (torch.arange(n, dtype=torch.float64) / n)).float()


def test_scaled_bands_are_their_formulas() -> None:
    bands = _bands()
    linear, one = rotary.scaled_bands(bands, 4.0, "linear")
    assert one == 1.0 and torch.allclose(linear, bands / 4, rtol=1e-6)
    ntk, one = rotary.scaled_bands(bands, 4.0, "ntk")
    base = 10000 * 4.0 ** (64 / 62)  # the base that the last band reaches the factor under
    assert one == 1.0 and torch.allclose(ntk, (1 / base ** (torch.arange(32, dtype=torch.float64) / 32)).float(), rtol=1e-5)
    assert ntk[0] == bands[0] and float(ntk[-1]) == pytest.approx(float(bands[-1]) / 4, rel=1e-6)
    yarn, amplitude = rotary.scaled_bands(bands, 4.0, "yarn", original_length=4096, slow=1, fast=32)
    assert amplitude == 0.1 * math.log(4.0) + 1
    turns = 4096 * bands.double() / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], bands[turns >= 32])
    assert torch.allclose(yarn[turns <= 1], bands[turns <= 1] / 4, rtol=1e-6)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((yarn < bands) & (yarn > bands / 4))[between].all()
    for method in rotary.SCALINGS:
        same, amplitude = rotary.scaled_bands(bands, 1.0, method)
        assert amplitude == 1.0 and torch.allclose(same, bands, rtol=1e-6)


def test_scaled_bands_refuse() -> None:
    for args in ((_bands(), 4.0, "other"), (_bands(), 0.5, "linear"), (_bands(), float("nan"), "ntk"),
                 (_bands().view(4, 8), 2.0, "ntk"), (_bands()[:0], 2.0, "ntk")):
        with pytest.raises(ValueError):
            rotary.scaled_bands(*args)
    with pytest.raises(ValueError):
        rotary.scaled_bands(_bands(), 4.0, "yarn", slow=32, fast=1)


def test_heads_and_tables_the_calls_refuse() -> None:
    q, table = torch.zeros(2, 5, 3, 16), torch.zeros(1, 5, 16)
    with pytest.raises(RuntimeError, match="HIP device"):
        rotary.rotary_forward(q, None, table)
    with pytest.raises(RuntimeError, match="HIP device"):
        rotary.rotary_backward(q, None, table)
    with pytest.raises(RuntimeError, match="HIP device"):
        rotary.rotary_table(torch.zeros(5, 1), _bands())
    with pytest.raises(ValueError, match="queries or keys"):
        rotary.rotary_forward(None, None, table)
    with pytest.raises(ValueError, match="layout"):
        rotary.rotary_forward(q, None, table, layout="other")
    with pytest.raises(TypeError):
        rotary.rotary_forward(q.double(), None, table)
    with pytest.raises(TypeError):
        rotary.rotary_forward(q, None, table.double())
    with pytest.raises(ValueError, match="heads"):
        rotary.rotary_forward(q[0], None, table)
    with pytest.raises(ValueError, match="heads"):
        rotary.rotary_forward(q, q[:, :4], table)
    with pytest.raises(ValueError, match="heads"):
        rotary.rotary_forward(q, q.bfloat16(), table)
    for bad in (table[:, :4], torch.zeros(3, 5, 16), torch.zeros(5)):
        with pytest.raises(ValueError, match="table"):
            rotary.rotary_forward(q, None, bad)
    for width in (15, 18):
        with pytest.raises(ValueError, match="rotary_dim"):
            rotary.rotary_forward(q, None, torch.zeros(1, 5, width))
    with pytest.raises(ValueError, match="head_dim"):
        rotary.rotary_forward(torch.zeros(2, 5, 3, 514), None, table)
    with pytest.raises(ValueError, match="norm weights"):
        rotary.rotary_forward(q, None, table, q_weight=torch.ones(8))
    with pytest.raises(ValueError, match="norm weights"):
        rotary.rotary_forward(q, q, table, q_weight=torch.ones(16), k_weight=torch.ones(16).bfloat16())
    with pytest.raises(ValueError, match="went in"):
        rotary.rotary_backward(q, None, table, q_weight=torch.ones(16))
    with pytest.raises(ValueError, match="one shape"):
        rotary.rotary_backward(q, None, table, q[:, :, :2], q_weight=torch.ones(16))
    with pytest.raises(RuntimeError, match="graph"):
        rotary.rotary_forward(q.clone().requires_grad_(), None, table)
    with pytest.raises(RuntimeError, match="no gradient for its table"):
        rotary.rotary(q, None, table.clone().requires_grad_())
    with pytest.raises(TypeError):
        rotary.rotary_table(torch.zeros(5, 1, dtype=torch.float64), _bands())
    with pytest.raises(ValueError):
        rotary.rotary_table(torch.zeros(5), _bands())


def _call(**fields):
    call = _native.MoRotaryCall()
    call.table, call.batch, call.tokens, call.head_dim, call.rotary_dim = 4096, 1, 4, 16, 16
    call.side[0].x = call.side[0].out = 4096
    call.side[0].heads = 2
    for name, value in fields.items():
        target = call.side[0] if hasattr(call.side[0], name) else call
        setattr(target, name, value)
    return call


def test_the_library_refuses_before_it_looks_for_a_device() -> None:
    lib = _native.load()
    for fields in ({"dtype": 3}, {"table_dtype": 3}, {"weight_dtype": 9}, {"batch": 0}, {"tokens": 0}, {"head_dim": 15},
                   {"head_dim": 514}, {"rotary_dim": 18}, {"rotary_dim": 0}, {"rotary_dim": 3}, {"table": 0},
                   {"table": 4097, "table_dtype": 2}, {"out": 0}, {"x": 0}, {"x": 4097}, {"heads": 0},
                   {"tokens": 1 << 30, "heads": 4}, {"batch": 1 << 31, "tokens": 2}):
        call = _call(**fields)
        assert lib.mo_rotary_forward(ctypes.byref(call), 0) == _native.MO_E_INVALID, fields
    for fields in ({"grad": 0}, {"grad": 4096, "weight": 4096}, {"grad": 4096, "weight": 4096, "x": 0},
                   {"grad": 4097}):
        call = _call(**fields)
        assert lib.mo_rotary_backward(ctypes.byref(call), 0, 0, 0) == _native.MO_E_INVALID, fields
    assert lib.mo_rotary_forward(None, 0) == _native.MO_E_INVALID
    assert lib.mo_rotary_table(0, 4096, 4096, 2, 1, 1, 1, 1.0, 0) == _native.MO_E_INVALID
    assert lib.mo_rotary_table(4096, 4096, 4096, 2, 1 << 31, 1, 1, 1.0, 0) == _native.MO_E_INVALID
    # the norm's partial sums: 16 fp16 values are one lane's, so 256 heads a workgroup, head_dim floats each
    call = _call(grad=4096, weight=4096, weight_grad=4096, tokens=1000)
    assert lib.mo_rotary_workspace_bytes(ctypes.byref(call)) == 8 * 16 * 4
