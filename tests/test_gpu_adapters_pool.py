"""Requests that have few adapters of a large pool, whose others hold anything: each form of the kernels against 64 bits."""

from __future__ import annotations

import pytest
import torch

from gpu_util import requires_gpu
from test_gpu_adapters import DTYPES, Case

pytestmark = requires_gpu

# rows, in, out, rank, where requests end, their adapters of nine
FORMS = [(50, 136, 104, 16, [0, 50], [7]), (50, 136, 104, 16, [3, 20, 20, 45], [7, 2, 7]), (33, 77, 51, 5, [0, 9, 33], [8, 0]),
         (60, 72, 88, 40, [0, 10, 30, 60], [4, -1, 100]), (1400, 72, 2056, 24, [0, 700, 1400], [1, 5]), (20, 2104, 64, 64, [0, 20], [3]),
         (8300, 104, 264, 32, [10, 5000, 8290], [6, 6]), (8300, 264, 104, 72, [0, 8300], [8])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,out,rank,cu,index", FORMS)
def test_few_of_many(rows, features, out, rank, cu, index, dtype) -> None:
    case = Case(rows, features, out, rank, dtype, count=9, cu=cu, index=index)
    for i in range(9):
        if i not in index:
            case.a[i], case.b[i] = float("nan"), float("inf")
    case.run()
    case.run(keep=True)
