"""Low-rank adapters of many requests on the GPU against 64 bits: ranks, odd sizes, ragged and empty requests, one adapter
twice, rows and requests without one, strides, the tokens in 8 bits, all gradients, by the formula and by differences."""

from __future__ import annotations

import pytest
import torch

from moss_offload import adapters
from moss_offload.kept8 import keep8

from gpu_util import requires_gpu
import kept8_model
from test_gpu_norm import _close, _randn

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0**-24
SPLIT = 2.0**-16  # what two bfloat16 parts of an fp32 number leave out, relative to it: half a step of a half step


class Case:
    def __init__(self, rows, features, out, rank, dtype, count=1, cu=None, index=None, tensor_scale=True, add=True, batch=None):
        self.x = _randn(rows, features, dtype=dtype)
        self.result, self.grad = _randn(rows, out, dtype=dtype, seed=1), _randn(rows, out, dtype=dtype, seed=2)
        self.a = (_randn(count, rank, features, seed=3) / features**0.5).to(dtype)
        self.b = _randn(count, out, rank, dtype=dtype, seed=4)
        self.scale = 0.5 + torch.rand(count, device=DEV) if tensor_scale else 0.75
        self.add = _randn(rows, features, dtype=dtype, seed=5) if add else None
        self.lead = (rows,) if batch is None else (batch, rows // batch)
        self.how = {"cu_seqlens": None if cu is None else torch.tensor(cu, device=DEV),
                    "index": None if index is None else torch.tensor(index, device=DEV)}
        requests = len(cu) - 1 if cu is not None else batch or 1
        bounds = cu if cu is not None else [i * (rows // requests) for i in range(requests + 1)]
        which = index if index is not None else [0] * requests if count == 1 else list(range(requests))
        self.pieces = [(bounds[i], bounds[i + 1], which[i]) for i in range(requests) if 0 <= which[i] < count]

    def shaped(self, t):
        return None if t is None else t.view(*self.lead, -1)

    def run(self, keep=False):
        y, hidden = adapters.adapters_forward(self.shaped(self.x), self.shaped(self.result), self.a, self.b, self.scale,
                                              hidden=True, **self.how)
        x, a, b, grad = (t.double() for t in (self.x, self.a, self.b, self.grad))
        read = kept8_model.read_back(self.x) if keep else x
        scale = self.scale.double() if isinstance(self.scale, torch.Tensor) else torch.full((len(a),), self.scale, device=DEV).double()
        rows, features, out, rank = x.shape[0], x.shape[1], b.shape[1], a.shape[1]
        h, dh = (torch.zeros(rows, rank, device=DEV, dtype=torch.float64) for _ in range(2))
        near_h, near_dh = torch.zeros_like(h), torch.zeros_like(dh)
        exact, near = self.result.double(), 3 * U * self.result.double().abs()
        dx = self.add.double() if self.add is not None else torch.zeros_like(x)
        near_dx = 3 * U * dx.abs()
        da, db = torch.zeros_like(a), torch.zeros_like(b)
        near_da, near_db = torch.zeros_like(a), torch.zeros_like(b)
        given = hidden.double()
        for low, high, i in self.pieces:
            p = slice(low, high)
            c = scale[i]
            # every sum: a rounding a term at most, the terms' products and a few around them; between the products
            # the numbers are fp32 or split in two
            h[p], near_h[p] = x[p] @ a[i].t(), (features + 8) * U * (x[p].abs() @ a[i].abs().t())
            exact[p] += c * (h[p] @ b[i].t())
            near[p] += c * (near_h[p] @ b[i].abs().t() + ((rank + 8) * U + SPLIT) * (h[p].abs() @ b[i].abs().t()))
            dh[p] = c * (grad[p] @ b[i])
            near_dh[p] = c * (out + 8) * U * (grad[p].abs() @ b[i].abs())
            dx[p] += dh[p] @ a[i]
            near_dx[p] += near_dh[p] @ a[i].abs() + ((rank + 8) * U + SPLIT) * (dh[p].abs() @ a[i].abs())
            da[i] += dh[p].t() @ read[p]
            near_da[i] += near_dh[p].t() @ read[p].abs() + ((rows + 8) * U + SPLIT) * (dh[p].abs().t() @ read[p].abs())
            db[i] += c * (grad[p].t() @ given[p])
            near_db[i] += c * ((rows + 8) * U + SPLIT) * (grad[p].abs().t() @ given[p].abs())
        _close(hidden, h, near_h, "hidden")
        _close(y.view(exact.shape), exact, near, "y")
        source = keep8(self.shaped(self.x)) if keep else self.shaped(self.x)
        call = (self.shaped(self.grad), source, hidden, self.a, self.b, self.scale)
        got = adapters.adapters_backward(*call, add=self.shaped(self.add), **self.how)
        _close(got[0].view(dx.shape), dx, near_dx, "dx")
        _close(got[1], da, near_da, "da")
        _close(got[2], db, near_db, "db")
        again = adapters.adapters_backward(*call, add=self.shaped(self.add), **self.how)
        assert all(torch.equal(s, t) for s, t in zip(got, again))
        assert torch.equal(adapters.adapters_forward(self.shaped(self.x), self.shaped(self.result), self.a, self.b, self.scale,
                                                     **self.how), y)


# rows, in, out, rank
SIZES = [(1, 1, 1, 1), (1, 64, 64, 16), (2, 33, 7, 3), (7, 100, 260, 5), (16, 256, 128, 8), (17, 96, 72, 13), (31, 520, 40, 16),
         (32, 64, 1032, 32), (65, 1001, 999, 33), (100, 384, 256, 64), (5, 72, 80, 100), (70, 200, 136, 128), (400, 128, 640, 16),
         (1300, 64, 96, 24), (300, 2056, 24, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("rows,features,out,rank", SIZES)
def test_sizes(rows, features, out, rank, keep, dtype) -> None:
    Case(rows, features, out, rank, dtype, tensor_scale=rank % 2 == 0, add=rank != 8).run(keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [4, 16, 40])
@pytest.mark.parametrize("cu,index", [
    ([0, 50], [1]), ([0, 20, 50], [2, 0]), ([0, 1, 2, 3, 50], [0, 1, 2, 1]), ([0, 0, 17, 17, 48, 48], [0, 1, 2, 1, 0]),
    ([3, 10, 45], [1, 1]), ([0, 50], [-1]), ([0, 10, 30, 50], [0, -1, 0]), ([0, 10, 30, 50], [3, 1 << 40, -(1 << 40)]),
    ([0, 0], [0]), ([50, 50], [2]), (list(range(51)), [i % 3 for i in range(50)]), ([0, 10, 30, 50], None)])
def test_requests(cu, index, rank, dtype) -> None:
    """Ragged and empty requests, an adapter twice or never, requests and rows without one."""

    for keep in (False, True):
        Case(50, 136, 104, rank, dtype, count=3, cu=cu, index=index).run(keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 64, 72, 128])
def test_long_requests(rank, dtype) -> None:
    """Tiles of 128 rows that share the weight, splits of the features, borders inside tiles."""

    for keep in (False, True):
        Case(4100, 4104, 4104, rank, dtype, count=2, cu=[3, 1500, 1500, 4000, 4090], index=[1, 0, 0, 1], add=keep).run(keep)
    Case(1100, 72, 2056, rank, dtype).run()


def test_the_same_in_one_launch_a_kernel_of_each_form() -> None:
    """Rows that are no multiple of anything, around the sizes where the form of a kernel changes."""

    for rows in (1023, 1024, 1025):
        for rank in (16, 40):
            Case(rows, 264, 1032, rank, torch.bfloat16, count=3, cu=[0, 300, 900, rows - 1], index=[2, 0, 1]).run()


def test_requests_by_batch() -> None:
    for dtype in DTYPES:
        Case(60, 72, 88, 8, dtype, count=4, batch=4).run()
        Case(60, 72, 88, 8, dtype, count=3, batch=5, index=[2, 0, 2, -1, 1]).run()
        Case(60, 72, 88, 8, dtype, count=1, batch=5).run(True)


def test_many_requests_and_long_ones() -> None:
    cuts = sorted({0, 2100, *(int(c) for c in torch.randint(0, 2100, (199,), generator=torch.Generator().manual_seed(1)))})
    index = [i % 7 for i in range(len(cuts) - 1)]
    Case(2110, 96, 72, 8, torch.bfloat16, count=7, cu=cuts, index=index).run(True)
    Case(5000, 64, 64, 16, torch.bfloat16, count=2, cu=[0, 1, 4096, 5000], index=[0, 1, 0]).run()
    Case(3, 4096, 2048, 16, torch.bfloat16, count=3, cu=[0, 1, 2, 3], index=[2, 0, 1]).run()
    Case(20, 9000, 300, 64, torch.bfloat16, count=2, cu=[0, 12, 20], index=[1, 0]).run()


def test_rows_behind_the_last_request_pass_the_result_on() -> None:
    case = Case(40, 64, 64, 8, torch.bfloat16, cu=[0, 30])
    case.x[30:], case.grad[30:] = float("nan"), float("nan")
    y, hidden = adapters.adapters_forward(case.x, case.result, case.a, case.b, 1.0, hidden=True, **case.how)
    assert torch.equal(y[30:], case.result[30:]) and torch.isfinite(y).all() and not hidden[30:].any()
    dx, da, db = adapters.adapters_backward(case.grad, case.x, hidden, case.a, case.b, 1.0, add=case.add, **case.how)
    assert torch.equal(dx[30:], case.add[30:]) and all(torch.isfinite(t).all() for t in (dx, da, db))


def test_wide_ranges() -> None:
    """Gradients far below and tokens far above one: nothing under- or overflows between the products."""

    for dtype, low, high in ((torch.bfloat16, 1e-20, 1e20), (torch.float32, 1e-20, 1e18), (torch.float16, 1e-6, 1e4)):
        case = Case(40, 96, 80, 16, dtype, tensor_scale=False)
        case.grad = (case.grad.float() * low).to(dtype)
        case.add = None
        case.run()
        case = Case(40, 96, 80, 16, dtype, tensor_scale=False)
        case.x = (case.x.float() * high).to(dtype)
        case.b = (case.b.float() / high).to(dtype)
        case.run()


def test_views_and_places() -> None:
    store = _randn(40, 900, dtype=torch.bfloat16)
    a, b = _randn(1, 8, 64, dtype=torch.bfloat16, seed=1), _randn(1, 96, 8, dtype=torch.bfloat16, seed=2)
    for x, result in ((store[:, :64], store[:, 64:160]), (store[:, 3:67], store[:, 101:197]), (store[:, :128:2], store[:, ::9][:, :96]),
                      (store[:1, :64].expand(40, -1), store[:, 200:296])):
        y, hidden = adapters.adapters_forward(x, result, a, b, hidden=True)
        plain, same = adapters.adapters_forward(x.contiguous(), result.contiguous(), a, b, hidden=True)
        # whole rows off the 16-byte grid may be summed in another order
        assert torch.allclose(hidden, same, rtol=1e-4, atol=1e-4) and torch.allclose(y.float(), plain.float(), rtol=2.0**-7, atol=1e-3)
        got = adapters.adapters_backward(result, x, hidden, a, b, add=x)
        want = adapters.adapters_backward(result.contiguous(), x.contiguous(), hidden, a, b, add=x.contiguous())
        for s, t in zip(got, want):
            assert torch.allclose(s.float(), t.float(), rtol=2.0**-7, atol=2.0**-8 * float(t.float().abs().max()))
    turned = adapters.adapters_forward(store[:, :64], store[:, 64:160], a.transpose(1, 2).contiguous().transpose(1, 2),
                                       b.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(turned, adapters.adapters_forward(store[:, :64], store[:, 64:160], a, b))


def test_no_rows() -> None:
    a, b = _randn(2, 4, 24), _randn(2, 40, 4)
    x, result, index = torch.empty(0, 24, device=DEV), torch.empty(0, 40, device=DEV), torch.tensor([1], device=DEV)
    y, hidden = adapters.adapters_forward(x, result, a, b, hidden=True, index=index)
    dx, da, db = adapters.adapters_backward(result, x, hidden, a, b, index=index)
    assert y.shape == (0, 40) and dx.shape == (0, 24) and not da.any() and not db.any()


def test_autograd_matches_the_calls_and_differences() -> None:
    x, result = _randn(3, 10, 24).requires_grad_(), _randn(3, 10, 40, seed=1).requires_grad_()
    a, b = _randn(2, 5, 24, seed=2).requires_grad_(), _randn(2, 40, 5, seed=3).requires_grad_()
    index = torch.tensor([1, -1, 0], device=DEV)
    grad, leaves = _randn(3, 10, 40, seed=4), [x, result, a, b]
    y = adapters.adapters(x, result, a, b, 0.5, index=index)
    got = torch.autograd.grad(y, leaves, grad)

    def value(x, result, a, b):
        out = result.clone()
        for i, which in enumerate(index.tolist()):
            if which >= 0:
                out[i] = out[i] + 0.5 * (x[i] @ a[which].t()) @ b[which].t()
        return (out * grad.double()).sum()

    wide = [t.detach().double() for t in leaves]
    for i, g in enumerate(got):
        way = _randn(*g.shape, seed=9 + i).double()
        up, down = ([v + (side * way if j == i else 0) for j, v in enumerate(wide)] for side in (0.5, -0.5))
        # the value is linear in each, so the difference is its slope; the gradients' terms sum to some 1e3 roundings
        assert abs(float((g.double() * way).sum() - (value(*up) - value(*down)))) <= 1e-4 * float((g.double() * way).abs().sum())


def test_autograd_shares_kept_tokens_and_skips_what_is_not_wanted() -> None:
    x = _randn(20, 64, dtype=torch.bfloat16).requires_grad_()
    result = _randn(20, 48, dtype=torch.bfloat16, seed=1)
    a, b = (_randn(8, 64, dtype=torch.bfloat16, seed=2).requires_grad_(), _randn(48, 8, dtype=torch.bfloat16, seed=3).requires_grad_())
    kept = keep8(x.detach())
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t), t)[1], lambda t: t):
        y = adapters.adapters(x, result, a, b, 2.0, keep=kept)
    assert any(t.data_ptr() == kept.values.data_ptr() for t in saved)
    assert not any(t.dtype == torch.bfloat16 and t.shape == x.shape for t in saved)
    grads = torch.autograd.grad(y, [x, a, b], torch.ones_like(y))
    own = torch.autograd.grad(adapters.adapters(x, result, a, b, 2.0, keep=True), [x, a, b], torch.ones_like(y))
    assert all(torch.equal(s, t) for s, t in zip(grads, own)) and grads[1].shape == a.shape
    for wanted in ([x], [a], [b]):
        leaves = [t if any(t is w for w in wanted) else t.detach() for t in (x, a, b)]
        y = adapters.adapters(leaves[0], result, leaves[1], leaves[2], 2.0, keep=True)
        (one,) = torch.autograd.grad(y, wanted, torch.ones_like(y))
        assert torch.equal(one, next(g for g, t in zip(grads, (x, a, b)) if t is wanted[0]))
    with torch.no_grad():
        assert not adapters.adapters(x, result, a, b).requires_grad
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(adapters.adapters(x, result, a, b).sum(), x, create_graph=True)


def test_refusals() -> None:
    x, result, a, b = _randn(6, 24), _randn(6, 40), _randn(2, 4, 24), _randn(2, 40, 4)
    index = torch.tensor([0], device=DEV)
    bad = [(x, result, a, b, 1.0, {}), (x, result[:5], a, b, 1.0, {"index": index}), (x, result, a[:, :, :23], b, 1.0, {"index": index}),
           (x, result, a, b[:, :39], 1.0, {"index": index}), (x, result, a.half(), b, 1.0, {"index": index}),
           (x, result, a, b, torch.ones(3, device=DEV), {"index": index}), (x, result, a, b, 1.0, {"index": index.float()}),
           (x, result, a, b, 1.0, {"index": index.expand(2)}), (x, result, a[0], b[0], 1.0, {}),
           (x, result, a, b, 1.0, {"index": index, "cu_seqlens": torch.tensor([0], device=DEV)}),
           (x, result, _randn(1, 129, 24), _randn(1, 40, 129), 1.0, {})]
    for *given, how in bad:
        with pytest.raises(ValueError):
            adapters.adapters_forward(*given, **how)
    with pytest.raises(RuntimeError):
        adapters.adapters_forward(x.requires_grad_(), result, a, b, index=index)
    x = x.detach()
    y, hidden = adapters.adapters_forward(x, result, a, b, index=index, hidden=True)
    for given in ((y[:5], x, hidden, a, b), (y, x[:5], hidden, a, b), (y, x, hidden[:5], a, b), (y, keep8(x[:, :23]), hidden, a, b),
                  (y, x, hidden.half(), a, b)):
        with pytest.raises(ValueError):
            adapters.adapters_backward(*given, index=index)
    with pytest.raises(ValueError):
        adapters.adapters(x, result, a, b, index=index, keep=keep8(x[:5]))
    with pytest.raises(RuntimeError, match="scales"):
        adapters.adapters(x, result, a, b, torch.ones(2, device=DEV, requires_grad=True), index=index)
