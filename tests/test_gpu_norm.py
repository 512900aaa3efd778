"""Norms on the GPU against 64 bits: both kinds, odd sizes, samples by batch and by lengths, rows in none, strides, the
input in 8 bits, all gradients, by the formula and by differences."""

from __future__ import annotations

import pytest
import torch

from moss_offload import norms
from moss_offload.kept8 import keep8

from gpu_util import requires_gpu
import kept8_model

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ROUNDING = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25, torch.float32: 2.0**-126}
U = 2.0**-24
ADDS = 44  # of a sum over a row: 16 a lane, 6 levels of a wave, 16 waves, and the products and the division around it


def _randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _close(got, exact, near, what=""):
    """``near``: what fp32 may be off by; then the rounding to the output's type."""

    dtype = got.dtype
    assert got.shape == exact.shape
    bound = near + ROUNDING[dtype] * (exact.abs() + near) + TINY[dtype]
    # to the nearest: a value past the type's largest by half a step or more is infinite (65504 + 16 for float16, whose
    # steps there are 32), so an infinity is right where the exact value with its error reaches that far
    past = torch.isinf(got) & (got.double().sign() * exact + near >= torch.finfo(dtype).max * (1 + ROUNDING[dtype] / 2))
    worst = torch.where(past, 0.0, (got.double() - exact).abs() / bound).max() if got.numel() else 0.0
    assert worst <= 1, (what, float(worst))


def _owner(rows, samples, cu):
    """[rows, samples] of zeros and ones."""

    if cu is None:
        return torch.eye(samples, device=DEV, dtype=torch.float64).repeat_interleave(rows // samples, 0)
    row = torch.arange(rows, device=DEV)[:, None]
    return ((row >= cu[:-1]) & (row < cu[1:])).double()


class Case:
    def __init__(self, rows, dim, dtype, kind, weight, bias, scale, shift, cu, lead=None, offset=0.0, wdtype=torch.float32):
        self.kind, self.cu, self.dtype = kind, cu, dtype
        samples = 0 if scale is None else scale
        self.x = (offset + _randn(rows, dim)).to(dtype)
        self.grad = _randn(rows, dim, dtype=dtype, seed=1)
        self.weight = (1 + 0.3 * _randn(dim, seed=2)).to(wdtype) if weight else None
        self.bias = (0.3 * _randn(dim, seed=3)).to(wdtype) if bias else None
        self.scale = (0.4 * _randn(samples, dim, seed=4)).to(dtype) if samples else None
        self.shift = (0.4 * _randn(samples, dim, seed=5)).to(dtype) if samples and shift else None
        self.lead = lead or ((samples, rows // samples) if samples and cu is None else (rows,))
        self.how = {"kind": kind, "scale": self.scale, "shift": self.shift, "cu_seqlens": cu}
        self.owner = _owner(rows, samples, cu) if samples else torch.ones(rows, 1, device=DEV, dtype=torch.float64)

    def shaped(self, t):
        return t.view(*self.lead, -1)

    def wide(self):
        dim = self.x.shape[1]
        one, zero = torch.ones(dim, device=DEV, dtype=torch.float64), torch.zeros(dim, device=DEV, dtype=torch.float64)
        w = one if self.weight is None else self.weight.double()
        b = zero if self.bias is None else self.bias.double()
        s = self.owner @ self.scale.double() if self.scale is not None else 0 * self.x.double()
        t = self.owner @ self.shift.double() if self.shift is not None else 0 * self.x.double()
        return w, b, s, t, self.owner.sum(1, keepdim=True)

    def check_forward(self, out, stats, eps=1e-6):
        w, b, s, t, live = self.wide()
        x = self.x.double()
        mean = x.mean(1, keepdim=True) if self.kind == "layer" else 0 * x[:, :1]
        r = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
        n = (x - mean) * r
        exact = ((n * w + b) * (1 + s) + t) * live
        # the mean: ADDS roundings of values as large as mean |x|; the square root takes half of the variance's
        # ADDS roundings and of twice the mean's error over the deviation
        off_mean = ADDS * U * x.abs().mean(1, keepdim=True) * r if self.kind == "layer" else 0 * r
        off = off_mean + n.abs() * ((ADDS / 2 + 6) * U + off_mean)
        near = w.abs() * (1 + s).abs() * off + 5 * U * ((n * w).abs() + b.abs()) * (1 + s.abs()) + 2 * U * t.abs()
        _close(out.view(x.shape), exact, near * live, "out")
        if stats is not None:
            _close(stats[:, 0], mean[:, 0], (off_mean / r)[:, 0], "mean")
            _close(stats[:, 1], r[:, 0], (r * ((ADDS / 2 + 6) * U + off_mean))[:, 0], "deviation")

    def check_backward(self, grads, stats, x):
        """From the statistics as given: ``x`` is what the kernel read, in 64 bits."""

        w, b, s, _, live = self.wide()
        rows, dim = self.x.shape
        mean, r = stats.double()[:, :1], stats.double()[:, 1:]
        n, g = (x - mean) * r, self.grad.double()
        h = g * (1 + s) * w * live
        size = g.abs() * (1 + s.abs()) * w.abs() * live  # what h's roundings are relative to
        along, level = (h * n).mean(1, keepdim=True), h.mean(1, keepdim=True) if self.kind == "layer" else 0 * r
        exact = r * (h - level - n * along)
        bound = size + n.abs() * (size * n.abs()).mean(1, keepdim=True)
        bound = bound + (size.mean(1, keepdim=True) if self.kind == "layer" else 0)
        _close(grads.x.view(x.shape), exact, (ADDS + 12) * U * r * bound, "dx")
        # sums over the rows: a rounding for each row at most, and those of the terms
        steps = (rows + 48) * U
        terms = {"weight": (live * (1 + s) * g * n, (1 + s.abs()) * (g * n).abs() * live),
                 "bias": (live * (1 + s) * g, (1 + s.abs()) * g.abs() * live)}
        for name, (term, large) in terms.items():
            got = getattr(grads, name)
            if got is not None:
                assert got.dtype == getattr(self, name).dtype
                _close(got, term.sum(0), steps * large.sum(0), name)
        if grads.scale is not None:
            _close(grads.scale, self.owner.t() @ (g * (n * w + b)),
                   steps * (self.owner.t() @ (g.abs() * ((n * w).abs() + b.abs()))), "scale")
        if grads.shift is not None:
            _close(grads.shift, self.owner.t() @ g, steps * (self.owner.t() @ g.abs()), "shift")
        for name in ("weight", "bias", "scale", "shift"):
            assert (getattr(grads, name) is None) == (getattr(self, name) is None)

    def run(self, keep=False):
        out, stats, kept = norms.norm_forward(self.shaped(self.x), self.weight, self.bias, stats=True, keep=keep, **self.how)
        self.check_forward(out, stats)
        plain = norms.norm_forward(self.shaped(self.x), self.weight, self.bias, **self.how)
        assert torch.equal(plain, out)
        source, x = self.shaped(self.x), self.x.double()
        if keep:
            values, exponents = kept8_model.keep(self.x)
            assert torch.equal(kept.values.view(values.shape), values)
            assert torch.equal(kept.exponents.view(exponents.shape), exponents)
            source, x = kept, kept8_model.read(values, exponents, x.shape[1])
        grads = norms.norm_backward(self.shaped(self.grad), source, stats, self.weight, self.bias, **self.how)
        self.check_backward(grads, stats, x)
        again = norms.norm_backward(self.shaped(self.grad), source, stats, self.weight, self.bias, **self.how)
        for first, second in zip(grads, again):
            assert first is second is None or torch.equal(first, second)


# rows, dim
SIZES = [(1, 1), (3, 2), (1, 7), (5, 8), (64, 31), (7, 100), (33, 511), (130, 512), (12, 520), (6, 1000), (9, 1024), (5, 1031),
         (20, 3072), (3, 4100), (4, 8192), (3, 8193), (2, 12288), (2, 16384), (2500, 64), (4200, 96), (3000, 1536)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("kind", norms.KINDS)
@pytest.mark.parametrize("rows,dim", SIZES)
def test_sizes(rows, dim, kind, keep, dtype) -> None:
    Case(rows, dim, dtype, kind, True, dim % 2 == 0, 1, True, None).run(keep)


@pytest.mark.parametrize("kind", norms.KINDS)
@pytest.mark.parametrize("weight,bias,scale,shift", [(0, 0, None, 0), (1, 0, None, 0), (0, 1, None, 0), (1, 1, None, 0),
                                                     (0, 0, 3, 1), (1, 0, 3, 0), (0, 1, 3, 1), (1, 1, 3, 1)])
def test_parts(weight, bias, scale, shift, kind) -> None:
    for keep in (False, True):
        Case(36, 200, torch.bfloat16, kind, weight, bias, scale, shift, None).run(keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cu", [[0, 1], [0, 40], [0, 7, 40], [0, 0, 3, 3, 3, 39, 39], [5, 9, 30], [0, 35], [0, 0], [40, 40, 40],
                                list(range(41)), [3, 3, 4, 4]])
def test_lengths(cu, dtype) -> None:
    """Empty samples, one row each, and rows before the first and behind the last: zeros, and part of no sum."""

    cu = torch.tensor(cu, device=DEV)
    case = Case(40, 72, dtype, "layer", True, True, cu.numel() - 1, True, cu)
    for keep in (False, True):
        case.run(keep)
    case.how["cu_seqlens"] = cu.int()
    case.run()


def test_long_lengths_over_many_workgroups() -> None:
    cuts = torch.tensor([0, 1, 700, 701, 2048, 2048, 4999, 5100], device=DEV)
    for dim in (40, 640):
        Case(5200, dim, torch.bfloat16, "rms", True, False, 7, True, cuts).run(True)
        Case(5200, dim, torch.float32, "layer", True, True, 7, True, cuts).run()


def test_many_samples() -> None:
    Case(3000, 48, torch.float32, "rms", True, True, 1500, True, None).run()


def test_rows_far_from_zero() -> None:
    """The squares are taken around the mean, so a large one costs its own roundings and no more."""

    for dtype in (torch.bfloat16, torch.float32):
        Case(10, 3072, dtype, "layer", True, True, None, False, None, offset=100.0).run()


@pytest.mark.parametrize("wdtype", DTYPES)
def test_types_of_weights(wdtype) -> None:
    Case(12, 96, torch.bfloat16, "layer", True, True, 1, True, None, wdtype=wdtype).run()


def test_views_and_places() -> None:
    store = _randn(9, 3, 700, dtype=torch.bfloat16)
    weight, scale = 1 + 0.1 * _randn(64), 0.1 * _randn(9, 6, 64, dtype=torch.bfloat16)
    for x in (store[..., :64], store[..., 3:67], store[..., ::2][..., :64], store[:, ::2, 8:72], store[:, :1, :64].expand(-1, 5, -1)):
        got, stats, _ = norms.norm_forward(x, weight, scale=scale[:, 1], shift=scale[:, 4], stats=True)
        want, other, _ = norms.norm_forward(x.contiguous(), weight, scale=scale[:, 1].contiguous(),
                                            shift=scale[:, 4].contiguous(), stats=True)
        assert torch.equal(got, want) and torch.equal(stats, other) and got.is_contiguous()
        grads = norms.norm_backward(x, x, stats, weight, scale=scale[:, 1], shift=scale[:, 4])
        again = norms.norm_backward(x.contiguous(), x.contiguous(), stats, weight, scale=scale[:, 1], shift=scale[:, 4])
        for a, b in zip(grads, again):
            assert a is b is None or torch.equal(a, b)


def test_no_rows() -> None:
    x, weight = torch.empty(0, 40, device=DEV), torch.ones(40, device=DEV)
    out, stats, kept = norms.norm_forward(x, weight, weight, stats=True, keep=True)
    assert out.shape == (0, 40) and stats.shape == (0, 2) and kept.shape == (0, 40)
    grads = norms.norm_backward(x, x, stats, weight, weight)
    assert grads.x.shape == (0, 40) and not grads.weight.any() and not grads.bias.any()


def test_not_finite_rows_stay_by_themselves() -> None:
    x = _randn(6, 96)
    x[1, 5], x[3, 40] = float("inf"), float("nan")
    out = norms.norm_forward(x)
    assert torch.isfinite(out[[0, 2, 4, 5]]).all() and torch.isnan(out[3]).all() and torch.isnan(out[1, 5])
    zero = norms.norm_forward(torch.zeros(2, 96, device=DEV), kind="layer")
    assert zero.eq(0).all()


def test_autograd_matches_the_calls_and_differences() -> None:
    x = _randn(2, 9, 40).requires_grad_()
    weight, bias = (1 + 0.2 * _randn(40, seed=1)).requires_grad_(), _randn(40, seed=2).requires_grad_()
    scale, shift = (0.2 * _randn(2, 40, seed=3)).requires_grad_(), _randn(2, 40, seed=4).requires_grad_()
    leaves = [x, weight, bias, scale, shift]
    grad = _randn(2, 9, 40, seed=5)
    for kind in norms.KINDS:
        out = norms.norm(x, weight, bias, kind=kind, scale=scale, shift=shift)
        got = torch.autograd.grad(out, leaves, grad)

        def value(*v):
            x, w, b, s, t = v
            c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
            n = c / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            return (((n * w + b) * (1 + s[:, None]) + t[:, None]) * grad.double()).sum()

        wide = [t.detach().double() for t in leaves]
        for i, g in enumerate(got):
            step = 1e-5
            way = _randn(*g.shape, seed=9 + i).double()
            up, down = ([v + (step * way if j == i else 0) * side for j, v in enumerate(wide)] for side in (1, -1))
            slope = (value(*up) - value(*down)) / (2 * step)
            # central differences are off by step^2 times a third derivative of order one; the gradients by 2^-20 of their terms
            assert abs(float((g.double() * way).sum() - slope)) <= 1e-5 * float((g.double() * way).abs().sum() + 1)


def test_autograd_asks_for_what_is_wanted_and_keeps_8_bits() -> None:
    x, weight = _randn(30, 64, dtype=torch.bfloat16).requires_grad_(), torch.ones(64, device=DEV)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append((t.dtype, t.shape)), t)[1], lambda t: t):
        out = norms.norm(x, weight, keep=True)
    assert (torch.bfloat16, x.shape) not in saved and (torch.int8, x.shape) in saved
    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
    _, stats, _ = norms.norm_forward(x.detach(), weight, stats=True)
    want = norms.norm_backward(torch.ones_like(out), keep8(x.detach()), stats, weight)
    assert torch.equal(dx, want.x)
    with torch.no_grad():
        assert not norms.norm(x, weight, keep=True).requires_grad
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(norms.norm(x, weight).sum(), x, create_graph=True)


def test_refusals() -> None:
    x, weight, scale = _randn(6, 40), torch.ones(40, device=DEV), torch.zeros(2, 40, device=DEV)
    with pytest.raises(ValueError):
        norms.norm_forward(x, kind="group")
    with pytest.raises(ValueError):
        norms.norm_forward(x, weight[:39])
    with pytest.raises(ValueError):
        norms.norm_forward(x, weight, weight.half())
    with pytest.raises(ValueError):
        norms.norm_forward(x, scale=scale)  # two samples, a first dimension of six
    with pytest.raises(ValueError):
        norms.norm_forward(x, cu_seqlens=torch.tensor([0, 6], device=DEV))
    with pytest.raises(ValueError):
        norms.norm_forward(x, scale=scale, cu_seqlens=torch.tensor([0, 6], device=DEV))
    with pytest.raises(ValueError):
        norms.norm_forward(x, scale=scale, cu_seqlens=torch.tensor([0, 2, 6]))
    with pytest.raises(ValueError):
        norms.norm_forward(torch.zeros(2, 16385, device=DEV))
    with pytest.raises(TypeError):
        norms.norm_forward(x.double())
    with pytest.raises(RuntimeError):
        norms.norm_forward(x.requires_grad_())
    x = x.detach()
    _, stats, _ = norms.norm_forward(x, stats=True)
    with pytest.raises(ValueError):
        norms.norm_backward(x, x[:5], stats)
    with pytest.raises(ValueError):
        norms.norm_backward(x, x, stats[:5])
    with pytest.raises(ValueError):
        norms.norm_backward(x, keep8(x.half()), stats)
