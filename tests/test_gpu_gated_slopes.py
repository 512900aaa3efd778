"""The gradients of saturated gates and ups, where the slopes are differences of numbers that round to one: within a few roundings of
their own size, against 64 bits."""

from __future__ import annotations

import pytest
import torch

from moss_offload import gated

from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0**-24
STEPS = 32  # roundings of fp32 on the way, each of the slope's or a term's own size


def _bend(x):
    """1 - tanh(x)^2 without a difference."""

    e = torch.exp(-2 * x.abs())
    return 4 * e / (1 + e).square()


def _check(got, exact, near, what):
    half = torch.finfo(got.dtype).eps / 2  # a rounding to the type; subnormals step by their own unit
    room = near + exact.abs() * half * 1.001 + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert torch.isfinite(got).all() and (got.double() - exact).abs().sub(room).max() <= 0, \
        (what, float(((got.double() - exact).abs() / room).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fused", [False, True])
def test_slopes_far_from_zero(fused, dtype) -> None:
    g = torch.cat((torch.linspace(-200, 200, 4001), torch.tensor([1e3, -1e3, 6e4, -6e4]))).to(DEV, dtype)
    for u in (torch.linspace(-2500, 2500, 4005, device=DEV).to(dtype), torch.linspace(-40, 40, 4005, device=DEV).to(dtype)):
        for scale in (1.0, 2.0**12):
            d = torch.full_like(u, scale)
            if fused:
                back = gated.gated_backward(d[None], torch.cat((u, g))[None])
                du, dg = back[0, :4005], back[0, 4005:]
            else:
                du, dg = (t[0] for t in gated.gated_backward(d[None], u[None], g[None]))
            wide_u, wide_g = u.double(), g.double()
            t, s, rest = torch.tanh(wide_g / 4), torch.sigmoid(wide_g), torch.sigmoid(-wide_g)
            exact = scale * 4 * t * s * _bend(wide_u / 25)
            first, second = _bend(wide_g / 4) * s, 4 * t * s * rest
            cap = scale * 25 * torch.tanh(wide_u / 25)
            # an exponential under the type's range is zero, and a product of some of them
            spare = 2.0**-112 * scale
            most = torch.finfo(dtype).max / 2
            here = (cap * (first + second)).abs() < most
            _check(du, exact, STEPS * U * exact.abs() + spare, "up")
            _check(dg[here], (cap * (first + second))[here], (STEPS * U * cap.abs() * (first + second.abs()) + spare)[here], "gate")
