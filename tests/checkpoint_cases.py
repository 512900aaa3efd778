"""Checkpoints whose input is kept in 8 bits under autocast, on whichever device: their parameters' gradients are those of the
same step without a checkpoint. Tokens are small whole numbers, which 8 bits keep as they are."""

from __future__ import annotations

import torch

from moss_offload.kept8 import checkpoint_kept8

WHERE = ["inside", "outside", "layer before", "layer after", "twice", "its own cast"]


def _step(where, device, checkpointed):
    torch.manual_seed(4)
    layers = torch.nn.Sequential(torch.nn.Linear(32, 32), torch.nn.GELU(), torch.nn.Linear(32, 32)).to(device)
    tokens = torch.randint(-60, 61, (6, 32), generator=torch.Generator().manual_seed(1)).float().to(device).requires_grad_()

    def block(t):
        if where != "its own cast":
            return layers(t)
        with torch.autocast(t.device.type, dtype=torch.bfloat16):
            return layers(t)

    def run(t):
        return checkpoint_kept8(block, t) if checkpointed else block(t)

    def loss():
        if where == "layer before":
            out = layers(tokens) + run(tokens)
        elif where == "layer after":
            out = layers(run(tokens))
        else:
            out = run(run(tokens)) if where == "twice" else run(tokens)
        return out.float().square().mean()

    if where == "its own cast":
        loss().backward()
    else:
        with torch.autocast(device.type, dtype=torch.bfloat16):
            value = loss()
            if where != "outside":
                value.backward()
        if where == "outside":
            value.backward()
    return [tokens.grad, *(p.grad for p in layers.parameters())]


def check(where, device) -> None:
    got, want = _step(where, device, True), _step(where, device, False)
    assert all(g is not None for g in got), [g is not None for g in got]
    for g, w in zip(got, want):
        if where == "twice":  # the second checkpoint's tokens are read back from 8 bits: some hundredths of them
            assert float((g - w).norm()) <= 0.1 * float(w.norm())
        else:  # the same products; parts of a gradient may be added in another order or rounded to bfloat16 once more
            assert float((g - w).norm()) <= 2.0**-7 * float(w.norm())
