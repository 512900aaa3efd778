"""8-bit floating-point linears on the GPU as a program calls them: biases of another type, no tokens and one, sums
that are exact, operands with room around them, saved columns that were offloaded, other strides."""

from __future__ import annotations

import pytest
import torch

from moss_offload import fp8_kernels as fp8

import fp8_model as model
from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _splits(rows, cols, reduction):
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    return [part["splits"] for part in fp8.product_plan(rows, cols, reduction, cus)]


# ---- biases ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,in_features,out_features,split", [(64, 128, 48, False), (300, 256, 272, False),
                                                                 (2, 3136, 64, True)])
@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, -8), (torch.float16, -11)])
def test_a_float32_bias_is_added_before_the_one_rounding(dtype, half, rows, in_features, out_features, split) -> None:
    """A product of 1 and a bias of a little over half a unit: the sum is past the tie, the bias alone rounds to it."""

    assert (max(_splits(rows, out_features, in_features)) > 1) == split
    weight, scale = fp8.fp8_quantize_weight(torch.ones(out_features, in_features, device=DEV))
    tokens = torch.zeros(rows, in_features, dtype=dtype, device=DEV)
    tokens[:, 5] = 1.0
    bias = torch.full((out_features,), 2.0**half + 2.0 ** (half - 12), device=DEV)
    exact = 1.0 + bias
    assert (exact.double() == 1.0 + bias.double()).all() and (exact.to(dtype) > 1.0 + 2.0**half).all()
    got = fp8.fp8_linear_forward(tokens, weight, scale, bias)
    assert got.dtype == dtype and torch.equal(got, exact.to(dtype).expand_as(got))
    assert torch.equal(fp8.fp8_linear(tokens, weight, scale, bias.requires_grad_()).detach(), got)


@pytest.mark.parametrize("rows", [1, 33, 300])
@pytest.mark.parametrize("bias_dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_bias_of_any_type(dtype, bias_dtype, rows) -> None:
    weight, scale = fp8.fp8_quantize_weight(0.02 * _randn(272, 400))
    tokens, bias = _randn(rows, 400, dtype=dtype, seed=1), _randn(272, seed=2).to(bias_dtype)
    a, b = model.read_back(tokens), model.decoded(weight, scale).t().contiguous()
    exact = a @ b + bias.double()
    one = torch.ones(rows, 1, device=DEV, dtype=torch.float64)
    bound = model.product_bound(dtype, torch.cat((a, one), 1), torch.cat((b, bias.double()[None]), 0), exact)
    got = fp8.fp8_linear_forward(tokens, weight, scale, bias)
    assert got.dtype == dtype and ((got.double() - exact).abs() <= bound).all()
