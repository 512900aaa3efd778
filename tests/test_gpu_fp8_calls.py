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


# ---- reading back ---------------------------------------------------------------------------------


def test_values_whose_rows_overlap_are_read_back() -> None:
    values, scales = fp8.fp8_quantize_rows(_randn(1, 272))
    want = fp8.fp8_decode(values, scales)
    spread = fp8.fp8_decode(values.expand(5, -1), scales.view(torch.uint8).expand(5, -1).view(fp8.E8M0))
    assert torch.equal(spread, want.expand(5, -1))
    line = values.view(272).as_strided((9, 144), (16, 1))
    got = fp8.fp8_decode(line, torch.ones(9, 2, device=DEV), dtype=torch.float32)
    assert torch.equal(got, line.float())


# ---- no tokens, and one ---------------------------------------------------------------------------


@pytest.mark.parametrize("lead", [(0,), (2, 0), ()])
@pytest.mark.parametrize("trained", [False, True])
def test_no_tokens_and_a_vector_have_gradients(trained, lead) -> None:
    tokens = _randn(*lead, 272, dtype=torch.bfloat16).requires_grad_()
    master, bias = (0.02 * _randn(144, 272)).requires_grad_(), _randn(144, seed=1).requires_grad_()
    weight, scale = fp8.fp8_quantize_weight(master.detach())
    y = fp8.fp8_linear(tokens, master, None, bias) if trained else fp8.fp8_linear(tokens, weight, scale, bias)
    wanted = [tokens, bias, *([master] if trained else [])]
    gradient = _randn(*lead, 144, dtype=torch.bfloat16, seed=2)
    grads = torch.autograd.grad(y, wanted, gradient)
    assert y.shape == (*lead, 144) and [g.shape for g in grads] == [t.shape for t in wanted]
    if lead:
        assert not any(g.any() for g in grads)
        return
    row, line = tokens.detach()[None], gradient[None]
    assert torch.equal(y.detach(), fp8.fp8_linear_forward(row, weight, scale, bias.detach())[0])
    assert torch.equal(grads[0], fp8.fp8_linear_backward(line, weight, scale)[0])
    assert torch.equal(grads[1], gradient.float())
    if trained:
        assert torch.equal(grads[2], fp8.fp8_weight_gradient(line, row))
    pair = fp8.fp8_quantize_rows(tokens.detach())
    assert torch.equal(fp8.fp8_linear_forward(pair, weight, scale, bias.detach(), dtype=torch.bfloat16), y.detach())
    assert torch.equal(fp8.fp8_decode(*pair).double(), model.read_back(row)[0])


def test_evaluation_gives_the_trained_forwards_bits() -> None:
    tokens, master = _randn(77, 272, dtype=torch.bfloat16), (0.02 * _randn(144, 272)).requires_grad_()
    with torch.no_grad():
        still = fp8.fp8_linear(tokens, master)
    assert torch.equal(still, fp8.fp8_linear(tokens, master).detach())


def test_a_graph_through_a_trained_weights_backward_is_refused() -> None:
    tokens, master = _randn(8, 272).requires_grad_(), (0.02 * _randn(144, 272)).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(fp8.fp8_linear(tokens, master).sum(), [tokens], create_graph=True)


# ---- sums -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,in_features,out_features", [
    (1, 3136, 512), (17, 512, 3136), (33, 144, 400), (65, 1152, 144), (130, 272, 1040), (300, 1552, 528), (515, 912, 1296),
    (1100, 256, 2064), (2050, 1296, 784)])
@pytest.mark.parametrize("kind", ["power", "float32"])
def test_sums_of_small_whole_numbers_are_exact(kind, rows, in_features, out_features) -> None:
    """Whole numbers up to 3: products up to 9 keep every bit in the e4m3 instructions (which drop what lies under
    2**-15 of the largest of neighbours), sums stay far under 2**24, so each output is its sum rounded once. One
    product lost or taken twice would show: fp32 scales of 1.5 times a power keep that."""

    g = torch.Generator(device="cuda").manual_seed(rows)

    def whole(*shape):
        return torch.randint(-3, 4, shape, device=DEV, generator=g).float()

    tokens, gradient, master = whole(rows, in_features), whole(rows, out_features), whole(out_features, in_features)
    weight, scale = fp8.fp8_quantize_weight(master)
    if kind == "float32":
        scale, master = scale.float() * 1.5, master * 1.5
    a, d, w = tokens.double(), gradient.double(), master.double()
    for dtype in DTYPES:
        assert torch.equal(fp8.fp8_linear_forward(tokens, weight, scale, dtype=dtype), (a @ w.t()).to(dtype))
        assert torch.equal(fp8.fp8_linear_backward(gradient, weight, scale, dtype=dtype), (d @ w).to(dtype))
        if kind == "power":
            assert torch.equal(fp8.fp8_weight_gradient(gradient, tokens, dtype=dtype), (d.t() @ a).to(dtype))
