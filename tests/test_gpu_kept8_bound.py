"""The bound of the 8-bit rule, on the kernels."""

from __future__ import annotations

import pytest
import torch

from moss_offload.kept8 import keep8

import kept8_bound
from gpu_util import requires_gpu

pytestmark = requires_gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_bound_and_its_ends(dtype) -> None:
    x = kept8_bound.groups(dtype, "cuda")
    kept8_bound.check(x, keep8(x).restore())
