"""Norms of a batch of no samples, whose modulation has no rows either: empty results, and zeros for what is summed."""

from __future__ import annotations

import pytest
import torch

from moss_offload import norms

from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", [(0, 7, 40), (0, 40)])
def test_no_samples(shape, packed, keep) -> None:
    x = torch.empty(shape, device=DEV, requires_grad=True)
    weight, bias = torch.ones(40, device=DEV, requires_grad=True), torch.zeros(40, device=DEV, requires_grad=True)
    scale, shift = (torch.empty(0, 40, device=DEV, requires_grad=True) for _ in range(2))
    cu = torch.zeros(1, dtype=torch.int64, device=DEV) if packed else None
    for kind in norms.KINDS:
        out = norms.norm(x, weight, bias, kind=kind, scale=scale, shift=shift, cu_seqlens=cu, keep=keep)
        assert out.shape == shape
        grads = torch.autograd.grad(out, [x, weight, bias, scale, shift], torch.empty_like(out))
        assert [g.shape for g in grads] == [t.shape for t in (x, weight, bias, scale, shift)]
        assert not grads[1].any() and not grads[2].any()


def test_rows_without_a_sample_to_be_in_are_refused() -> None:
    scale = torch.empty(0, 40, device=DEV)
    with pytest.raises(ValueError):
        norms.norm_forward(torch.zeros(3, 40, device=DEV), scale=scale)
    with pytest.raises(ValueError):
        norms.norm_forward(torch.zeros(3, 40, device=DEV), scale=scale, cu_seqlens=torch.zeros(1, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):  # two samples of no rows, a modulation of none
        norms.norm_forward(torch.zeros(2, 0, 40, device=DEV), scale=scale)
