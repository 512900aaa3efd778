"""The bound of the 8-bit rule, on its model."""

from __future__ import annotations

import pytest
import torch

import kept8_bound
import kept8_model


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_bound_and_its_ends(dtype) -> None:
    x = kept8_bound.groups(dtype, "cpu")
    kept8_bound.check(x, kept8_model.read_back(x))
