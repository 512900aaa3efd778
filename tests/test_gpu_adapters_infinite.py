"""Infinite tokens and gradients under the adapters: infinities where the definition has them, whatever the rank is padded to."""

from __future__ import annotations

import pytest
import torch

from moss_offload import adapters

from gpu_util import requires_gpu
from test_gpu_norm import _randn

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# the forward pass in one launch and in two, split features, tiles of 128 rows, sizes that are no multiples of eight
FORMS = [(16, 64, 80, 8), (5, 256, 1032, 24), (20, 64, 80, 40), (40, 128, 72, 4), (33, 77, 51, 13), (50, 2104, 2056, 24), (1400, 48, 3080, 8),
         (8300, 104, 264, 24), (8300, 104, 264, 72)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,out,rank", FORMS)
def test_infinities_stay_infinities(rows, features, out, rank, dtype) -> None:
    """a is positive and a column of b has one sign, so no sum meets infinities of both."""

    x, result = _randn(rows, features, dtype=dtype), _randn(rows, out, dtype=dtype, seed=1)
    a = (_randn(1, rank, features, seed=2).abs() + 0.1).to(dtype)
    sign = torch.where(torch.arange(out, device=DEV) % 3 == 0, -1.0, 1.0)
    b = ((_randn(1, out, rank, seed=3).abs() + 0.1) * sign[:, None]).to(dtype)
    x[rows // 2, features // 3], x[rows - 1, 0] = float("inf"), float("-inf")
    y, hidden = adapters.adapters_forward(x, result, a, b, 0.5, hidden=True)
    assert torch.isinf(hidden).any(1).nonzero().flatten().tolist() == [rows // 2, rows - 1]
    assert torch.equal(hidden[rows // 2], torch.full_like(hidden[0], float("inf"))) and hidden[-1].eq(float("-inf")).all()
    assert y[rows // 2].double().eq(float("inf") * sign).all() and y[-1].double().eq(float("-inf") * sign).all()
    others = [i for i in range(rows) if i not in (rows // 2, rows - 1)]
    assert torch.isfinite(y[others]).all()

    grad = _randn(rows, out, dtype=dtype, seed=4)
    grad[0, 1], grad[rows // 3, out - 1] = float("inf"), float("-inf")
    dx, _, _ = adapters.adapters_backward(grad, x, hidden, a, b.abs(), 0.5)
    assert dx[0].eq(float("inf")).all() and dx[rows // 3].eq(float("-inf")).all()
    assert torch.isfinite(dx[[i for i in range(rows) if i not in (0, rows // 3)]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out,rank", [(16, 80, 8), (16, 80, 16), (40, 1032, 16), (1400, 3080, 16), (33, 72, 24), (2100, 264, 32), (31, 51, 13)])
def test_an_infinite_weight_gives_an_infinity(rows, out, rank, dtype) -> None:
    """h has all of its 24 bits, so that no part of it is zero."""

    g = torch.Generator(device="cuda").manual_seed(rows)
    n = torch.randint(1 << 23, 1 << 24, (rows, rank), device=DEV, generator=g) | 0x8001
    x, a = torch.zeros(rows, 3 * rank, device=DEV, dtype=dtype), torch.zeros(1, rank, 3 * rank, device=DEV, dtype=dtype)
    for i, mask in enumerate((0xFF0000, 0xFF00, 0xFF)):
        x[:, i::3] = ((n & mask).double() * 2.0**-24).to(dtype)
        a[0, range(rank), range(i, 3 * rank, 3)] = 1.0
    b = _randn(1, out, rank, dtype=dtype, seed=1)
    b[0, 3, rank - 1], b[0, out - 1, 0] = float("inf"), float("-inf")
    y = adapters.adapters_forward(x, torch.zeros(rows, out, device=DEV, dtype=dtype), a, b)
    assert y[:, 3].eq(float("inf")).all() and y[:, out - 1].eq(float("-inf")).all()
    assert torch.isfinite(y[:, [i for i in range(out) if i not in (3, out - 1)]]).all()
