"""Weights in training in 8-bit floating point under the activation offload hooks: the tokens' columns and their scales
go to host memory and come back in a layout of their own."""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

from moss_offload import dit, fp8_kernels, get_engine
from oracle import reference_hooks

from gpu_util import requires_gpu
from test_gpu_dit_fp8 import _model, _step

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


class _Trained(nn.Module):
    def __init__(self, linear: nn.Linear):
        super().__init__()
        self.weight = linear.weight

    def forward(self, tokens):
        return fp8_kernels.fp8_linear(tokens, self.weight)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("checkpointing", [False, True])
def test_offloaded_training_step_is_the_resident_one(checkpointing, packed) -> None:
    base = _model(torch.bfloat16)
    names = dit.joint_linear_names(base)
    for name in names:
        dit._replace(base, name, _Trained(base.get_submodule(name)))
    # the conditions of packed tokens are gathered, and torch sums a gather's gradient by atomics: what lies behind
    # it does not repeat from step to step, with or without offload
    for name, parameter in base.named_parameters():
        parameter.requires_grad_(name.removesuffix(".weight") in names)
    base.gradient_checkpointing = checkpointing
    offloaded = copy.deepcopy(base)
    offloaded.activation_offload = True
    want, want_grads = _step(base, packed)
    engine = get_engine(DEV)
    before = engine.stats()["bytes_unpacked"]
    got, grads = _step(offloaded, packed)
    assert engine.stats()["bytes_unpacked"] > before
    assert reference_hooks.bitwise_equal(got, want)
    assert grads.keys() == want_grads.keys() == {f"{name}.weight" for name in names}
    for name in grads:
        assert reference_hooks.bitwise_equal(grads[name], want_grads[name]), name


@pytest.mark.parametrize("rows", [1, 13, 77, 300])
def test_columns_come_back_from_the_host(rows) -> None:
    """The scales of 272 columns in three groups of tokens are laid group by group, and dense when they return."""

    g = torch.Generator(device="cuda").manual_seed(rows)
    tokens = torch.randn(rows, 272, device=DEV, generator=g).bfloat16()
    master = 0.02 * torch.randn(144, 272, device=DEV, generator=g)
    gradient = torch.randn(rows, 144, device=DEV, generator=g).bfloat16()

    def step():
        leaves = tokens.clone().requires_grad_(), master.clone().requires_grad_()
        return torch.autograd.grad(fp8_kernels.fp8_linear(*leaves), leaves, gradient)

    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    for a, b in zip(got, want):
        assert reference_hooks.bitwise_equal(a, b)
