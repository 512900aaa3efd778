"""Blocks on an 8-bit floating-point base swapped to host memory, against the resident model."""

from __future__ import annotations

import copy

import pytest
import torch

from moss_offload import dit
from moss_offload.memory import place_model

from gpu_util import assert_bitwise, requires_gpu
from test_gpu_dit_fp8 import _model, _step

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("rotary", ["composed", "hip"])
@pytest.mark.parametrize("mode", ["sync", "async"])
def test_swapped_blocks_give_the_resident_step(mode, rotary) -> None:
    base = _model(torch.bfloat16, layers=4)
    dit.quantize_joint_linears_fp8(base)
    dit.inject_lora(base, rank=4, alpha=4.0)
    dit.configure_rotary(base, rotary)
    base.gradient_checkpointing = True
    swapped = copy.deepcopy(base).cpu()
    place_model(swapped, DEV, 3, block_swap_mode=mode)
    try:
        want, want_grads = _step(base)
        for _ in range(2):
            got, grads = _step(swapped)
            assert_bitwise(got, want)
            assert grads.keys() == want_grads.keys()
            for name in grads:
                assert_bitwise(grads[name].to(DEV), want_grads[name])
    finally:
        if swapped.block_swap_manager is not None:
            swapped.block_swap_manager.close()
    last = swapped.layers[3].proj["q"].base
    assert last.weight_fp8.dtype == torch.float8_e4m3fn and last.weight_scale.dtype == torch.float8_e8m0fnu
