"""``checkpoint_kept8`` under autocast on the GPU."""

from __future__ import annotations

import pytest
import torch

import checkpoint_cases
from gpu_util import requires_gpu

pytestmark = requires_gpu


@pytest.mark.parametrize("where", checkpoint_cases.WHERE)
def test_parameters_keep_their_gradients(where) -> None:
    checkpoint_cases.check(where, torch.device("cuda", 0))
