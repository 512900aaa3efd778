"""Infinite and undefined gates and ups, by the definition: where the results are undefined and what they are elsewhere."""

from __future__ import annotations

import pytest
import torch

from moss_offload import gated

from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_situ_at_infinities_and_nan(dtype) -> None:
    g = torch.tensor([[INF, -INF, NAN, 1.0, INF, 2.0, NAN, 3.0]], device=DEV, dtype=dtype)
    u = torch.tensor([[1.0, 1.0, 1.0, INF, -INF, NAN, INF, -INF]], device=DEV, dtype=dtype)
    out = gated.gated_forward(u, g)
    assert torch.isnan(out)[0].tolist() == [False, False, True, False, False, True, True, False]
    assert out[0, 1] == 0 and out[0, 4] == -100.0
    gate = 4 * torch.tanh(g.double() / 4) * torch.sigmoid(g.double())
    exact = gate * 25 * torch.tanh(u.double() / 25)
    known = ~torch.isnan(exact)
    assert torch.equal(known, ~torch.isnan(out))
    # 32 roundings of fp32 and one to the type
    assert ((out.double() - exact)[known].abs() <= (32 * 2.0**-24 + torch.finfo(dtype).eps / 2) * exact[known].abs()).all()
    du, dg = gated.gated_backward(torch.ones_like(u), u, g)
    # a saturated gate or up has no slope
    assert torch.isnan(du)[0].tolist() == torch.isnan(dg)[0].tolist() == [False, False, True, False, False, True, True, False]
    assert dg[0, [0, 1, 4]].eq(0).all() and du[0, [1, 3, 4, 7]].eq(0).all()
