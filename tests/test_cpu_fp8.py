"""What the 8-bit floating-point calls refuse, on the CPU: no call here reaches a GPU."""

from __future__ import annotations

import pytest
import torch

from moss_offload import _native, fp8_kernels as fp8

import fp8_model as model


def _weight(out_features=32, in_features=144):
    scale = torch.full((-(-out_features // 128), -(-in_features // 128)), 127, dtype=torch.uint8)
    return torch.zeros(out_features, in_features).to(torch.float8_e4m3fn), scale.view(torch.float8_e8m0fnu)


def test_model_rounds_as_the_format_does() -> None:
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(model.round_e4m3(every), every)
    between = torch.linspace(-448, 448, 100_001).double()  # float32 numbers: one rounding on either side
    assert torch.equal(model.round_e4m3(between), between.float().to(torch.float8_e4m3fn).double())
    assert model.power_for(torch.tensor([448.0, 448.001, 0.0, 224.0, 2.0**-140], dtype=torch.float64)).tolist() == \
        [0, 1, -126, -1, -126]


def test_matrices_the_quantizers_refuse() -> None:
    for call in (fp8.fp8_quantize_rows, fp8.fp8_quantize_columns, fp8.fp8_quantize_both, fp8.fp8_quantize_weight):
        with pytest.raises(RuntimeError, match="HIP device"):
            call(torch.zeros(32, 64))
        with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
            call(torch.zeros(32, 64, dtype=torch.float64))
        with pytest.raises(ValueError, match="multiple"):
            call(torch.zeros(32, 24))
        with pytest.raises(ValueError, match="multiple"):
            call(torch.zeros(32, 0))
        with pytest.raises(RuntimeError, match="graph"):
            call(torch.zeros(32, 64, requires_grad=True))
    for shape in ((2, 32, 64), (0, 64)):
        with pytest.raises(ValueError, match="matrix, not empty"):
            fp8.fp8_quantize_weight(torch.zeros(shape))


def test_operands_the_products_refuse() -> None:
    weight, scale = _weight()
    tokens = torch.zeros(4, 144, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="float8_e4m3fn matrix"):
        fp8.fp8_linear_forward(tokens, weight.float(), scale)
    with pytest.raises(RuntimeError, match="float8_e4m3fn matrix"):
        fp8.fp8_linear_forward(tokens, weight.t(), scale)
    for bad in (scale[:, :1], scale.view(torch.uint8), scale.float().half(), scale.float().t()):
        with pytest.raises(RuntimeError, match="weight scale"):
            fp8.fp8_linear_forward(tokens, weight, bad)
    with pytest.raises(ValueError, match="144 features"):
        fp8.fp8_linear_forward(tokens[:, :128], weight, scale)
    with pytest.raises(ValueError, match="32 features"):
        fp8.fp8_linear_backward(tokens, weight, scale)
    with pytest.raises(RuntimeError, match="HIP device"):
        fp8.fp8_linear_forward(tokens, weight, scale)
    with pytest.raises(RuntimeError, match="HIP device"):
        fp8.fp8_linear_backward(tokens[:, :32], weight, scale)
    with pytest.raises(RuntimeError, match="HIP device"):
        fp8.fp8_weight_gradient(tokens[:, :32], tokens)
    with pytest.raises(ValueError, match="same rows"):
        fp8.fp8_weight_gradient(tokens[:3, :32], tokens)
    values, scales = weight[:, :144], torch.zeros(32, 2).to(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="one scale"):
        fp8.fp8_linear_forward((values, scales[:, :1]), weight, scale)
    with pytest.raises(RuntimeError, match="float8_e4m3fn of 144"):
        fp8.fp8_linear_forward((values.float(), scales), weight, scale)
    with pytest.raises(TypeError, match="two matrices or two quantized pairs"):
        fp8.fp8_weight_gradient((values, scales), tokens)
    with pytest.raises(ValueError, match="number of tokens"):
        fp8.fp8_weight_gradient((values, scales), (values, scales))
    with pytest.raises(TypeError):
        fp8.fp8_decode(values.float(), scales)
    with pytest.raises(ValueError, match="cols"):
        fp8.fp8_decode(values, scales, cols=145)
    with pytest.raises(ValueError, match="do not fit"):
        fp8.fp8_decode(values, scales[:5])


def test_the_library_refuses_before_it_looks_for_a_device() -> None:
    lib = _native.load()
    quantize = [4096, 1, 4, 64, 64, 4096, 4096, 0, 0, 0]
    for index, value, message in [(0, 0, b"null"), (1, 3, b"type"), (2, 0, b"empty"), (3, 24, b"multiples"),
                                  (4, 32, b"stride"), (4, 68, b"aligned"), (0, 4100, b"aligned"), (6, 0, b"pairs"),
                                  (2, 1 << 31, b"rows")]:
        call = list(quantize)
        call[index] = value
        assert lib.mo_fp8_quantize(*call) == _native.MO_E_INVALID
        assert message in lib.mo_last_error(), (index, value, lib.mo_last_error())
    forward = [4096, 0, 1, 4, 64, 64, 4096, 4096, 0, 32, 0, 4096, 1, 4096, 1 << 20, 0]
    for index, value, message in [(6, 0, b"null"), (8, 2, b"scale type"), (4, 40, b"multiples"), (9, 0, b"empty"),
                                  (11, 0, b"null"), (12, 5, b"type"), (11, 4104, b"misaligned"), (3, 0, b"empty")]:
        call = list(forward)
        call[index] = value
        assert lib.mo_fp8_linear_forward(*call) == _native.MO_E_INVALID
        assert message in lib.mo_last_error(), (index, value, lib.mo_last_error())
    call = list(forward)
    call[4], call[5], call[9] = 1 << 16, 1 << 16, 1 << 15  # 2^31 values
    assert lib.mo_fp8_linear_forward(*call) == _native.MO_E_INVALID and b"too large" in lib.mo_last_error()
    assert lib.mo_fp8_workspace_bytes(_native.MO_FP8_FORWARD, 0, 64, 64, 0, 0, 1) == 0
    weight = [4096, 0, 1, 32, 4096, 0, 1, 64, (1 << 23) - 127, 64, 32, 4096, 2, 4096, 1 << 40, 0]
    assert lib.mo_fp8_weight_gradient(*weight) == _native.MO_E_INVALID and b"too many rows" in lib.mo_last_error()


def test_plans_cover_the_reduction() -> None:
    """Every split has work, and few rows or long reductions are shared out while large calls are not."""

    for rows in (1, 77, 333, 1333, 4608, 17792, (1 << 31) - 1):
        for cols, reduction in ((3072, 3072), (16, 17792), (24576, 3072), (3072, 24576), (80, 128), (16, 16)):
            for cus in (32, 256):
                for floats in (False, True):
                    for dtype in (torch.bfloat16, torch.float32):
                        plan = fp8.product_plan(rows, cols, reduction, cus, float_scales=floats, dtype=dtype)
                        steps = -(-reduction // 128)
                        assert sum(part["rows"] for part in plan) == rows
                        for part in plan:
                            assert part["edge"] in (64, 128, 256) and 1 <= part["splits"] <= 32
                            covered = part["splits"] * part["split_steps"]
                            assert covered - part["split_steps"] < steps <= covered
                            if part["splits"] > 1:
                                assert part["split_steps"] >= 2 and part["splits"] * part["rows"] * cols * 4 <= 1 << 31
                        if len(plan) == 2:  # whole rounds of large tiles first
                            assert plan[0]["edge"] == 256 and plan[0]["splits"] == 1 and plan[0]["rows"] % 256 == 0
    assert fp8.product_plan(1, 3072, 12288, 256)[0]["splits"] > 1
    assert fp8.product_plan(4608, 24576, 3072, 256) == [{"rows": 4608, "edge": 256, "splits": 1, "split_steps": 24}]
    assert [part["rows"] for part in fp8.product_plan(17792, 3072, 12288, 256)] == [16384, 1408]


@pytest.mark.parametrize("rows", [1, 5, 16, 17])
@pytest.mark.parametrize("spare", [0, 2])
def test_tight_scales_are_laid_out_again(rows, spare):
    from moss_offload import fp8_kernels

    room = torch.arange(rows + spare, dtype=torch.uint8).add(100)
    tight = room.view(torch.float8_e8m0fnu)[:rows].unsqueeze(1)
    values = torch.zeros(rows, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = fp8_kernels._pair((values, tight), 128, "tokens")[1]
    assert scales.untyped_storage().nbytes() - scales.storage_offset() >= -(-rows // 16) * 16
    assert torch.equal(scales.view(torch.uint8), tight.view(torch.uint8))
