"""Activations in 8 bits by the rule, in 64 bits: what the kernels have to give bit for bit."""

from __future__ import annotations

import torch

GROUP = 32


def _steps(device) -> torch.Tensor:
    """2**-126 to 2**122, exact: a library's power need not be."""

    return torch.tensor([2.0**e for e in range(-126, 123)], dtype=torch.float64, device=device)


def keep(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, exponents)`` of a floating tensor ``[..., cols]``."""

    cols = x.shape[-1]
    wide = torch.nn.functional.pad(x.double(), (0, -cols % GROUP)).unflatten(-1, (-1, GROUP))
    peak = wide.abs().amax(-1)
    finite = torch.isfinite(wide).all(-1)
    steps = _steps(x.device)
    index = torch.searchsorted(127.0 * steps, torch.where(finite, peak, torch.zeros_like(peak)))
    step = steps[index]
    values = torch.round(wide / step.unsqueeze(-1))
    most = torch.where(64.0 * step > torch.finfo(x.dtype).max, 63.0, 127.0).unsqueeze(-1)
    values = torch.where(finite.unsqueeze(-1), torch.minimum(torch.maximum(values, -most), most), torch.zeros_like(values))
    exponents = torch.where(finite, index + 1, torch.full_like(index, 255))
    return values.flatten(-2).to(torch.int8), exponents.to(torch.uint8)


def read(values: torch.Tensor, exponents: torch.Tensor, cols: int) -> torch.Tensor:
    """The values in 64 bits; NaN where the exponent is 255."""

    step = _steps(exponents.device)[(exponents.long() - 1).clamp(0, 248)]
    step = torch.where(exponents == 255, torch.nan, step)
    return (values.double().unflatten(-1, (-1, GROUP)) * step.unsqueeze(-1)).flatten(-2)[..., :cols]


def read_back(x: torch.Tensor) -> torch.Tensor:
    return read(*keep(x), x.shape[-1])
