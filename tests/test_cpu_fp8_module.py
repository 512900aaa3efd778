"""``FrozenFp8Linear`` moved and cast, on the CPU."""

from __future__ import annotations

import pytest
import torch

from moss_offload import dit

FORMATS = (torch.float8_e4m3fn, torch.float8_e8m0fnu), (torch.float8_e4m3fn, torch.float32)


def _module(scale_dtype, device="cpu"):
    return dit.FrozenFp8Linear(torch.ones(32, 144, device=device).to(torch.float8_e4m3fn),
                               torch.ones(1, 2, device=device).to(scale_dtype), torch.float32)


def _formats(module):
    return module.weight_fp8.dtype, module.weight_scale.dtype


@pytest.mark.parametrize("formats", FORMATS)
def test_a_move_keeps_what_it_made(formats) -> None:
    """What a move makes of the buffers is what the module holds: nothing is moved a second time from the old ones."""

    module = _module(formats[1])
    made = []
    module._apply(lambda t: made.append(t.clone()) or made[-1])
    assert any(module.weight_fp8 is t for t in made) and any(module.weight_scale is t for t in made)
    assert _formats(module) == formats and module.compute_dtype == torch.float32


@pytest.mark.parametrize("formats", FORMATS)
def test_a_module_without_memory_is_given_some(formats) -> None:
    module = _module(formats[1], "meta").to_empty(device="cpu")
    assert module.weight_fp8.device.type == module.weight_scale.device.type == "cpu"
    module.load_state_dict(_module(formats[1]).state_dict())
    assert _formats(module) == formats and (module.weight_fp8.float() == 1).all()


@pytest.mark.parametrize("formats", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_cast_changes_the_compute_type_alone(dtype, formats) -> None:
    module = _module(formats[1])
    weight, scale = module.weight_fp8.clone(), module.weight_scale.clone()
    module.to(dtype)
    assert _formats(module) == formats and module.compute_dtype == dtype
    assert torch.equal(module.weight_fp8.view(torch.uint8), weight.view(torch.uint8))
    assert torch.equal(module.weight_scale.float(), scale.float())
