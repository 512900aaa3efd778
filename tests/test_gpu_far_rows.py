"""The block's kernels on rows whose distances, and on batches whose sizes, pass 32 bits, bit for bit against rows side by
side. What they are at ordinary distances is tested against 64 bits elsewhere.
"""

from __future__ import annotations

import pytest
import torch

from moss_offload import adapters, gated, kept8, norms

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _apart(rows: torch.Tensor, stride: int) -> torch.Tensor:
    """The same rows, ``stride`` elements apart."""

    room = torch.empty((len(rows) - 1) * stride + rows.shape[1], dtype=rows.dtype, device=DEV)
    view = room.as_strided(rows.shape, (stride, 1))
    view.copy_(rows)
    return view


def _randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


def _same(got, want):
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("dim", [200, 77])
def test_norms(dim) -> None:
    x, grad, weight, scale = _randn(3, dim), _randn(3, dim, seed=1), _randn(dim, seed=2), _randn(1, dim, seed=3)

    def run(x, grad):
        out, stats, _ = norms.norm_forward(x, weight, scale=scale, stats=True)
        return out, stats, *(g for g in norms.norm_backward(grad, x, stats, weight, scale=scale) if g is not None)

    _same(run(_apart(x, (1 << 31) + 8), _apart(grad, (1 << 31) + 16)), run(x, grad))


@pytest.mark.parametrize("cols", [200, 77])
def test_gated(cols) -> None:
    up, gate, grad = _randn(3, cols), _randn(3, cols, seed=1), _randn(3, cols, seed=2)

    def run(up, gate, grad):
        out, *kept = gated.gated_forward(up, gate, keep=True)
        return out, *(t for k in kept for t in (k.values, k.exponents)), *gated.gated_backward(grad, up, gate)

    _same(run(*(_apart(t, (1 << 31) + 8) for t in (up, gate, grad))), run(up, gate, grad))


@pytest.mark.parametrize("cols", [200, 77])
def test_kept(cols) -> None:
    x = _randn(3, cols)
    far, near = kept8.keep8(_apart(x, (1 << 31) + 8)), kept8.keep8(x)
    _same((far.values, far.exponents), (near.values, near.exponents))


@pytest.mark.parametrize("rank", [16, 32, 12])
@pytest.mark.parametrize("requests", [1, 600])
def test_adapters(rank, requests) -> None:
    rows, features, out, stride = 1200, 72, 200, 1 << 22  # the last row begins past 2^32 elements
    x, result, grad = _randn(rows, features), _randn(rows, out, seed=1), _randn(rows, out, seed=2)
    a, b = _randn(2, rank, features, seed=3), _randn(2, out, rank, seed=4)
    index = torch.arange(requests, device=DEV) % 2
    how = {"cu_seqlens": torch.arange(requests + 1, device=DEV) * (rows // requests), "index": index}

    def run(x, result, grad):
        y, hidden = adapters.adapters_forward(x, result, a, b, 0.5, hidden=True, **how)
        return y, hidden, *adapters.adapters_backward(grad, x, hidden, a, b, 0.5, **how)

    want = run(x, result, grad)
    for far in (0, 1, 2):  # one at a time: 10 GB each
        _same(run(*(_apart(t, stride) if i == far else t for i, t in enumerate((x, result, grad)))), want)
