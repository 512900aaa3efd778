"""The adapters' and norms' kernels for thousands of rows against 64 bits, with borders inside their tiles, and the sizes at
which a kernel's form changes."""

from __future__ import annotations

import pytest
import torch

import test_gpu_adapters
import test_gpu_norm

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [24, 32, 64, 72, 128])
def test_adapters(rank, dtype) -> None:
    for keep in (False, True):
        test_gpu_adapters.Case(8200, 136, 264, rank, dtype, count=2, cu=[3, 1500, 1500, 7000, 8190], index=[1, 0, 0, 1],
                               add=keep).run(keep)
    test_gpu_adapters.Case(8192, 520, 72, rank, dtype).run()


@pytest.mark.parametrize("rows", [8191, 8192, 8193])
def test_adapters_around_a_change_of_form(rows) -> None:
    for rank in (16, 32):
        test_gpu_adapters.Case(rows, 72, 136, rank, torch.bfloat16, count=3, cu=[0, 300, 900, rows - 1], index=[2, 0, 1]).run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [2048, 2049, 2056, 3580, 3584, 3592, 4096])
def test_norms(dim, dtype) -> None:
    cuts = torch.tensor([2, 500, 500, 1203, 1300], device="cuda:0")
    for keep in (False, True):
        test_gpu_norm.Case(1303, dim, dtype, "layer", True, True, 4, True, cuts).run(keep)
    test_gpu_norm.Case(2, dim, dtype, "rms", True, False, 1, True, None).run()
