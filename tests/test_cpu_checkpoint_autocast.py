"""``checkpoint_kept8`` under autocast on the CPU, its kernels and the device's random numbers' state replaced by the model of the
8-bit rule."""

from __future__ import annotations

import pytest
import torch

from moss_offload import kept8

import checkpoint_cases
import kept8_model


@pytest.mark.parametrize("where", checkpoint_cases.WHERE)
def test_parameters_keep_their_gradients(where, monkeypatch) -> None:
    monkeypatch.setattr(kept8, "keep8", lambda t: kept8.Kept8(*kept8_model.keep(t.detach()), t.shape[-1], t.dtype))
    monkeypatch.setattr(kept8.Kept8, "restore",
                        lambda self: kept8_model.read(self.values, self.exponents, self.cols).to(self.dtype))
    monkeypatch.setattr(torch.cuda, "get_rng_state", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "set_rng_state", lambda state, device=None: None)
    checkpoint_cases.check(where, torch.device("cpu"))
