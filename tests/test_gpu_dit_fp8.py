"""The DiT on an 8-bit floating-point base with fused rotary positions: a LoRA step, with and without offload,
against the same model on the composed operations and on the definition of the 8-bit linear."""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

from moss_offload import dit, fp8_kernels, get_engine
from oracle import reference_hooks

import fp8_model
from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


def _model(dtype=torch.float32, layers=2):
    torch.manual_seed(0)
    model = dit.MOSSImageTransformer(dim=128, ffn_dim=256, num_heads=4, num_layers=layers, text_dim=32, freq_dim=16,
                                     latent_channels=16)
    dit.init_weights(model, std=0.05)
    return model.to(DEV, dtype).train()


def _step(model, packed=False):
    g = torch.Generator(device="cuda").manual_seed(1)
    dtype = model.compute_dtype
    latents = torch.randn(2, 16, 6, 5, device=DEV, generator=g).to(dtype)
    context = torch.randn(2, 7, 32, device=DEV, generator=g).to(dtype)
    timestep = torch.tensor([300.0, 800.0], device=DEV)
    model.zero_grad(set_to_none=True)
    if packed:
        out = torch.stack(model.forward_packed(list(latents), timestep, list(context)))
    else:
        out = model(latents, timestep, context)
    out.float().square().mean().backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters() if p.requires_grad}
    return out.detach().clone(), grads


def _near(a, b, bound):
    off = float((a.double() - b.double()).norm() / b.double().norm())
    assert off <= bound, off


class _DefinedLinear(nn.Module):
    """The 8-bit linear by its definition in 64 bits, differentiable as the kernels are."""

    def __init__(self, weight, scale):
        super().__init__()
        self.register_buffer("decoded", fp8_model.decoded(weight, scale))
        self.out_features, self.in_features = weight.shape

    @property
    def weight(self):
        return torch.empty(0, device=self.decoded.device)

    class _Function(torch.autograd.Function):
        @staticmethod
        def forward(ctx, tokens, decoded):
            ctx.save_for_backward(decoded)
            rows = tokens.reshape(-1, tokens.shape[-1])
            return (fp8_model.read_back(rows) @ decoded.t()).to(tokens.dtype).view(*tokens.shape[:-1], -1)

        @staticmethod
        def backward(ctx, gradient):
            (decoded,) = ctx.saved_tensors
            rows = gradient.reshape(-1, gradient.shape[-1])
            return (fp8_model.read_back(rows) @ decoded).to(gradient.dtype).view(*gradient.shape[:-1], -1), None

    def forward(self, tokens):
        return self._Function.apply(tokens, self.decoded)


@pytest.mark.parametrize("packed", [False, True])
def test_fused_rotary_gives_the_composed_step(packed) -> None:
    """float32 throughout: the same function, rounded once instead of at every operation."""

    composed = _model()
    fused = copy.deepcopy(composed)
    assert dit.configure_rotary(fused, "hip") == 4
    want, want_grads = _step(composed, packed)
    got, grads = _step(fused, packed)
    _near(got, want, 2.0**-14)
    assert grads.keys() == want_grads.keys()
    for name in grads:
        if want_grads[name].norm() > 0:
            _near(grads[name], want_grads[name], 2.0**-10)
    assert any("q_norm" in name and want_grads[name].norm() > 0 for name in grads)


def test_step_on_an_fp8_base_is_the_definitions() -> None:
    """A step of one 8-bit value is 2**-4 of it; two runs whose sums differ in the last bits of fp32 step apart at
    a few of the thousands of values that a block rounds, so the whole differs by far less than one step."""

    base = _model()
    names = dit.quantize_joint_linears_fp8(base)
    assert len(names) == 2 * 6
    defined = copy.deepcopy(base)
    for name in names:
        module = defined.get_submodule(name)
        dit._replace(defined, name, _DefinedLinear(module.weight_fp8, module.weight_scale))
    torch.manual_seed(3)
    dit.inject_lora(base, rank=4, alpha=4.0)
    for name in names:
        wrapped = dit.LoRALinear(defined.get_submodule(name), 4, 4.0).to(DEV)
        wrapped.load_state_dict({k: v for k, v in base.get_submodule(name).state_dict().items() if "lora" in k}, strict=False)
        dit._replace(defined, name, wrapped)
    for model in (base, defined):
        for name, parameter in model.named_parameters():
            parameter.requires_grad_("lora_" in name)
    want, want_grads = _step(defined)
    got, grads = _step(base)
    _near(got, want, 2.0**-6)
    assert len(grads) == 24
    for name in grads:
        _near(grads[name], want_grads[name], 2.0**-4)


@pytest.mark.parametrize("checkpointing", [False, True])
def test_offloaded_step_is_the_resident_one(checkpointing) -> None:
    """bfloat16, fp8 base, fused rotary, LoRA: the offloaded saves come back as they went."""

    base = _model(torch.bfloat16)
    dit.quantize_joint_linears_fp8(base)
    dit.inject_lora(base, rank=4, alpha=4.0)
    dit.configure_rotary(base, "hip")
    base.gradient_checkpointing = checkpointing
    offloaded = copy.deepcopy(base)
    offloaded.activation_offload = True
    want, want_grads = _step(base)
    got, grads = _step(offloaded)
    assert reference_hooks.bitwise_equal(got, want)
    for name in grads:
        assert reference_hooks.bitwise_equal(grads[name], want_grads[name]), name
    assert get_engine(DEV).stats()["bytes_unpacked"] > 0


def test_module_keeps_its_formats_and_its_state() -> None:
    linear = nn.Linear(144, 64, bias=False).to(DEV)
    module = dit.FrozenFp8Linear.from_weight(linear.weight)
    assert module.compute_dtype == torch.float32
    module.to(torch.bfloat16)
    assert module.compute_dtype == torch.bfloat16
    assert module.weight_fp8.dtype == torch.float8_e4m3fn and module.weight_scale.dtype == torch.float8_e8m0fnu
    tokens = torch.randn(3, 5, 144, device=DEV)
    want = fp8_kernels.fp8_linear_forward(tokens.bfloat16(), module.weight_fp8, module.weight_scale)
    assert torch.equal(module(tokens), want)
    again = dit.FrozenFp8Linear(torch.zeros_like(module.weight_fp8), module.weight_scale.clone(), torch.bfloat16)
    again.load_state_dict(module.state_dict())
    assert torch.equal(again(tokens), want)


def test_training_every_weight_in_8_bits() -> None:
    """fp8_linear on a master weight: a few steps of gradient descent bring a linear fit down."""

    g = torch.Generator(device="cuda").manual_seed(5)
    target = torch.randn(64, 128, device=DEV, generator=g)
    weight = torch.zeros(64, 128, device=DEV, requires_grad=True)
    losses = []
    for step in range(40):
        tokens = torch.randn(256, 128, device=DEV, generator=g)
        loss = (fp8_kernels.fp8_linear(tokens, weight) - tokens @ target.t()).square().mean()
        losses.append(float(loss))
        (grad,) = torch.autograd.grad(loss, weight)
        with torch.no_grad():
            weight -= 16.0 * grad
    assert losses[-1] < 0.02 * losses[0], losses


def test_rotary_backend_names() -> None:
    with pytest.raises(ValueError, match="rotary backend"):
        dit.configure_rotary(nn.Module(), "other")
