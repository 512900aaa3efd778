"""How far a value may be from what 8 bits keep of it, at the ends of the types and of a step."""

from __future__ import annotations

import torch


def groups(dtype, device) -> torch.Tensor:
    """``[groups, 32]``: peaks around 63.5 and 127 steps, from the type's smallest numbers to its largest, beside values all over."""

    info = torch.finfo(dtype)
    g = torch.Generator().manual_seed(5)
    steps = [2.0**e for e in range(-126, 122) if info.smallest_normal / 64 <= 2.0**e <= info.max / 128]
    peaks = [p * s for s in steps for p in (63.5, 63.51, 63.75, 64.0, 96.3, 126.9, 127.0, 127.01) if p * s <= info.max]
    peaks += [info.max, info.max * 0.999, info.max * 0.9971, info.max * 0.99, info.smallest_normal, info.smallest_normal * info.eps,
              info.smallest_normal / 4, 0.0]
    x = torch.tensor(peaks, dtype=torch.float64)[:, None] * (2 * torch.rand(len(peaks), 32, generator=g, dtype=torch.float64) - 1)
    x[:, 3] = torch.tensor(peaks, dtype=torch.float64)
    x[:, 9], x[:, 17] = -x[:, 3], x[:, 3] * 0.996
    x = x.to(dtype)
    return x[torch.isfinite(x).all(1)].to(device)


def check(x, back) -> None:
    wide, back = x.double(), back.double()
    off, peak = (back - wide).abs(), wide.abs().amax(1, keepdim=True)
    held = peak > 63 * torch.finfo(x.dtype).max / 64  # only there can a value be past 63 of a step whose 64 is past the type
    assert torch.isfinite(back).all()
    assert (off <= torch.where(held, peak / 64, (peak / 127).clamp(min=2.0**-127))).all()
    # and no less than that: 2**-7 of the largest is passed, by more where values are held
    assert (off > peak * 2.0**-7).any()
    most = off[:, 3] > peak[:, 0] / 127 * 1.0001
    assert held[most & (peak[:, 0] > 2.0**-120), 0].all()
    assert (most & held[:, 0]).any()
