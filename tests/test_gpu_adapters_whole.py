"""The numbers between the adapters' products keep all of their 24 bits: differences of neighbours, which nothing but the last of
them make, come out exact. Each form of the kernels."""

from __future__ import annotations

import pytest
import torch

from moss_offload import adapters
from moss_offload.kept8 import keep8

from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
UNIT = 2.0**-24


def _numbers(*shape, dim, seed):
    """Whole numbers of 24 bits, of which neighbours along ``dim`` (2i, 2i + 1) differ by 1 to 255: in units of 2**-24 they
    and every partial sum of them are exact in fp32, and the differences in every type."""

    g = torch.Generator(device="cuda").manual_seed(seed)
    n = torch.randint(1 << 23, (1 << 24) - 256, shape, device=DEV, generator=g).movedim(dim, 0)
    n[1::2] = n[:-1:2] + torch.randint(1, 256, n[1::2].shape, device=DEV, generator=g)
    return n.movedim(0, dim)


def _parts(n, features, dtype):
    """``[rows, features]``: the number of rank j as eight bits each in the columns 3 j to 3 j + 2."""

    out = torch.zeros(n.shape[0], features, device=DEV, dtype=torch.float64)
    for i, mask in enumerate((0xFF0000, 0xFF00, 0xFF)):
        out[:, i : 3 * n.shape[1] : 3] = (n & mask).double() * UNIT
    return out.to(dtype)


def _ones(rank, features, dtype):
    """``[rank, features]``: what adds a rank's three columns up."""

    out = torch.zeros(rank, features, device=DEV, dtype=dtype)
    for i in range(3):
        out[range(rank), range(i, 3 * rank, 3)] = 1.0
    return out


def _apart(count, other, dtype):
    """``[count, other]``: in column c, 1 and -1 at two neighbours."""

    out = torch.zeros(count, other, device=DEV, dtype=dtype)
    column = torch.arange(other, device=DEV)
    pair = column % (count // 2)
    out[2 * pair, column], out[2 * pair + 1, column] = 1.0, -1.0
    return out


# rows, the features of the reduced side, the other side's, rank, where requests end: the forward pass in one launch and in two, split
# features, tiles of 128 rows, sizes that are no multiples of eight
FORMS = [(16, 48, 40, 16, None), (21, 200, 72, 10, (5, 6, 21)), (40, 128, 1032, 32, None), (33, 200, 136, 64, (0, 30)), (50, 2104, 2056, 16, None),
         (9, 4104, 520, 64, None), (1400, 48, 3080, 16, (3, 700, 1390)), (8300, 104, 264, 32, (10, 5000, 8290)), (8200, 208, 136, 64, None),
         (8200, 392, 136, 128, None), (70, 400, 72, 128, None), (31, 77, 35, 13, None), (50, 101, 99, 32, (0, 50)), (2100, 1032, 24, 24, None)]


def _how(rows, cu):
    return ({}, torch.ones(rows, dtype=torch.bool, device=DEV)) if cu is None else (
        {"cu_seqlens": torch.tensor(cu, device=DEV), "index": torch.zeros(len(cu) - 1, dtype=torch.int64, device=DEV)},
        (torch.arange(rows, device=DEV) >= cu[0]) & (torch.arange(rows, device=DEV) < cu[-1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,reduced,other,rank,cu", FORMS)
def test_forward(rows, reduced, other, rank, cu, dtype) -> None:
    n = _numbers(rows, rank, dim=1, seed=rows)
    how, inside = _how(rows, cu)
    result = torch.zeros(rows, other, device=DEV, dtype=dtype)
    y, hidden = adapters.adapters_forward(_parts(n, reduced, dtype), result, _ones(rank, reduced, dtype)[None],
                                          _apart(rank, other, dtype).t()[None], hidden=True, **how)
    n = torch.where(inside[:, None], n, torch.zeros_like(n))
    assert torch.equal(hidden.double(), n.double() * UNIT)
    pair = torch.arange(other, device=DEV) % (rank // 2)
    assert torch.equal(y.double(), (n[:, 2 * pair] - n[:, 2 * pair + 1]).double() * UNIT)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,reduced,other,rank,cu", FORMS)
def test_input_gradient(rows, reduced, other, rank, cu, dtype) -> None:
    n = _numbers(rows, rank, dim=1, seed=rows + 1)
    how, inside = _how(rows, cu)
    x, hidden = torch.zeros(rows, other, device=DEV, dtype=dtype), torch.zeros(rows, rank, device=DEV)
    dx, _, _ = adapters.adapters_backward(_parts(n, reduced, dtype), x, hidden, _apart(rank, other, dtype)[None],
                                          _ones(rank, reduced, dtype).t()[None], **how)
    n = torch.where(inside[:, None], n, torch.zeros_like(n))
    pair = torch.arange(other, device=DEV) % (rank // 2)
    assert torch.equal(dx.double(), (n[:, 2 * pair] - n[:, 2 * pair + 1]).double() * UNIT)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("rows,reduced,other,rank,cu", FORMS)
def test_weight_gradients(rows, reduced, other, rank, cu, keep, dtype) -> None:
    rows -= rows % 2
    n = _numbers(rows, rank, dim=0, seed=rows + 2)
    how, inside = _how(rows, None if cu is None else (*cu[:-1], min(cu[-1], rows)))
    pair = torch.arange(other, device=DEV) % (rows // 2)
    inside = inside.long()
    want = n[2 * pair] * inside[2 * pair, None] - n[2 * pair + 1] * inside[2 * pair + 1, None]
    # a pair that a request's end parts leaves one number, which is rounded to the type
    want = (want.double() * UNIT).to(dtype)
    both = _apart(rows, other, dtype)
    x = keep8(both) if keep else both
    zero = torch.zeros(rows, rank, device=DEV)
    a, b = torch.zeros(1, rank, other, device=DEV, dtype=dtype), _ones(rank, reduced, dtype).t()[None]
    _, da, _ = adapters.adapters_backward(_parts(n, reduced, dtype), x, zero, a, b, **how)
    assert torch.equal(da[0].t(), want)
    x = torch.zeros(rows, 16, device=DEV, dtype=dtype)
    a, b = torch.zeros(1, rank, 16, device=DEV, dtype=dtype), torch.zeros(1, other, rank, device=DEV, dtype=dtype)
    _, _, db = adapters.adapters_backward(both, x, (n.double() * UNIT).float(), a, b, **how)
    assert torch.equal(db[0], want)
