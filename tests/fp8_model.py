"""The 8-bit floating-point definitions in 64 bits, for the tests: groups of 128, power-of-two scales, e4m3.

Written from the format: an e4m3 number has four significant bits down to 2**-6 and steps of 2**-9 below, at
most 448; a group's scale is the smallest power of two, from 2**-126 on, that brings it within 448.
"""

from __future__ import annotations

import torch

GROUP = 128


def power_for(peak: torch.Tensor) -> torch.Tensor:
    """The scale's exponent for groups of largest magnitude ``peak`` (finite, float64)."""

    exponents = torch.arange(-126, 121, device=peak.device)
    powers = torch.tensor([2.0**int(e) for e in exponents], dtype=torch.float64, device=peak.device)
    return exponents[(peak.unsqueeze(-1) <= 448.0 * powers).to(torch.uint8).argmax(-1)]


def two_to(exponent: torch.Tensor) -> torch.Tensor:
    table = torch.tensor([2.0**i for i in range(-160, 160)], dtype=torch.float64, device=exponent.device)
    return table[exponent.long() + 160]


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    step = torch.full_like(v, 2.0**-9)
    for i in range(-6, 9):
        step[v.abs() >= 2.0**i] = 2.0 ** (i - 3)
    return torch.round(v / step) * step


def row_groups(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(values, exponents) of a matrix in groups of 128 along its rows, values under their scales."""

    rows, cols = x.shape
    padded = torch.nn.functional.pad(x.double(), (0, -cols % GROUP)).view(rows, -1, GROUP)
    exponent = power_for(padded.abs().amax(-1))
    values = round_e4m3(padded / two_to(exponent).unsqueeze(-1))
    return values.flatten(1)[:, :cols], exponent


def block_groups(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    rows, cols = x.shape
    padded = torch.nn.functional.pad(x.double(), (0, -cols % GROUP, 0, -rows % GROUP))
    blocks = padded.view(-(-rows // GROUP), GROUP, -(-cols // GROUP), GROUP)
    exponent = power_for(blocks.abs().amax((1, 3)))
    values = round_e4m3(blocks / two_to(exponent)[:, None, :, None])
    return values.reshape(padded.shape)[:rows, :cols], exponent


def spread(values: torch.Tensor, shape) -> torch.Tensor:
    """One number a block of 128 x 128, repeated over ``shape``."""

    wide = values.repeat_interleave(GROUP, 0)[: shape[0]]
    return wide.repeat_interleave(GROUP, 1)[:, : shape[1]]


def read_back(x: torch.Tensor) -> torch.Tensor:
    values, exponent = row_groups(x)
    return values * two_to(exponent).repeat_interleave(GROUP, 1)[:, : x.shape[1]]


def decoded(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return weight.double() * spread(scale.double(), weight.shape)


# Half a unit in the last place of each output type (8, 11 and 24 significant bits), relative to a normal number.
ROUNDING = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
SMALLEST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24, torch.float32: 2.0**-126}


def product_bound(dtype: torch.dtype, a: torch.Tensor, b: torch.Tensor, exact: torch.Tensor) -> torch.Tensor:
    """How far a product of decoded operands ``a @ b`` may be from ``exact``: the last rounding, and sums.

    fp32 sums of n products: at most n 2**-24 of the sum of their magnitudes (each addition rounds a
    partial sum that is no larger). The e4m3 matrix instructions, which the 16-bit outputs come from, also drop
    bits under 2**-15 of the largest of up to 16 neighbouring products from each of them: at most 16 *
    2**-15 of that largest one, which is at most 2**-11 of their magnitudes' sum.
    """

    magnitude = a.abs() @ b.abs()
    sums = (a.shape[1] + 2) * 2.0**-24 + (0.0 if dtype == torch.float32 else 2.0**-11)
    near = sums * magnitude
    return near + ROUNDING[dtype] * (exact.abs() + near) + SMALLEST[dtype]
