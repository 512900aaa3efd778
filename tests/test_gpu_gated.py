"""Gated activations on the GPU against 64 bits: both kinds, odd sizes, fused and apart, strides, in 8 bits, values at the
ends, and the gradients by the formula and by differences."""

from __future__ import annotations

import pytest
import torch

from moss_offload import dit, gated
from moss_offload.kept8 import Kept8

from gpu_util import requires_gpu
import kept8_model
from test_gpu_norm import _close, _randn

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0**-24
# fp32 roundings of an output: an exponential's argument and value, a sum, a reciprocal or division, two series or
# quotients for the hyperbolic tangents, each within a few units, and the products: fewer than 32 in all
STEPS = 32


def _value(u, g, kind):
    if kind == "silu":
        return u * g * torch.sigmoid(g)
    return 4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(u / 25)


def _check(out, u, g, kind):
    exact = _value(u, g, kind)
    # an exponential past the type's range makes the sigmoid zero where it is under 2^-120
    _close(out, exact, STEPS * U * exact.abs() + 2.0**-112 * (1 + u.abs()) * (1 + g.abs()))


def _check_backward(du, dg, d, u, g, kind):
    s = torch.sigmoid(g)
    if kind == "silu":
        act, cap, slope, cap_slope = g * s, u, s * (1 + g * (1 - s)), torch.ones_like(u)
        size = s * (1 + g.abs())
    else:
        t, c = torch.tanh(g / 4), torch.tanh(u / 25)
        act, cap, cap_slope = 4 * t * s, 25 * c, 1 - c * c
        slope, size = (1 - t * t) * s + 4 * t * s * (1 - s), 5 * s  # both differences are of numbers up to 1
    spare = 2.0**-112 * (1 + d.abs()) * (1 + u.abs()) * (1 + g.abs())
    _close(du, d * act * cap_slope, STEPS * U * (d * act).abs() + spare, "up")
    _close(dg, d * cap * slope, STEPS * U * (d * cap).abs() * size + spare, "gate")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", gated.KINDS)
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 32), (5, 33), (17, 100), (64, 1024), (9, 1001), (300, 40)])
def test_forward_and_backward_match_64_bits(rows, cols, fused, keep, kind, dtype) -> None:
    both = (3 * _randn(rows, 2 * cols)).to(dtype)
    u, g = both[:, :cols], both[:, cols:]
    d = _randn(rows, cols, dtype=dtype, seed=1)
    given = (both, None) if fused else (u, g)
    out = gated.gated_forward(*given, kind=kind)
    _check(out, u.double(), g.double(), kind)
    source, (wide_u, wide_g) = given, (u.double(), g.double())
    if keep:
        again, *source = gated.gated_forward(*given, kind=kind, keep=True)
        assert torch.equal(again, out)
        pairs = [kept8_model.keep(t) for t in (u, g)]
        for i, (values, exponents) in enumerate(pairs):
            got = (source[0].values[:, i], source[0].exponents[:, i]) if fused else (source[i].values, source[i].exponents)
            assert torch.equal(got[0], values) and torch.equal(got[1], exponents)
        wide_u, wide_g = (kept8_model.read(*p, cols) for p in pairs)
    back = gated.gated_backward(d, *source, kind=kind)
    du, dg = (back[:, :cols], back[:, cols:]) if fused else back
    _check_backward(du, dg, d.double(), wide_u, wide_g, kind)


@pytest.mark.parametrize("kind", gated.KINDS)
def test_every_bfloat16(kind) -> None:
    """Each finite pattern as a gate and as an up, small, large and past the exponential's range."""

    bits = torch.arange(1 << 16, device=DEV, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    bits = bits[torch.isfinite(bits)]
    for dtype in (torch.bfloat16, torch.float32):
        sweep = bits.to(dtype)
        for other in (0.0, 1e-3, -0.7, 3.0, -40.0, 200.0):
            fixed = torch.full_like(sweep, other)
            for u, g in ((sweep, fixed), (fixed, sweep)):
                if kind == "silu":  # a product past the type's range is infinite in both
                    keep = (u.double() * g.double()).abs() < 1e38
                    u, g = u[keep], g[keep]
                out = gated.gated_forward(u[None], g[None], kind=kind)
                _check(out, u[None].double(), g[None].double(), kind)
                d = torch.full_like(u, 0.5)
                du, dg = gated.gated_backward(d[None], u[None], g[None], kind=kind)
                _check_backward(du, dg, d[None].double(), u[None].double(), g[None].double(), kind)


def test_views_and_places() -> None:
    store = _randn(6, 5, 400, dtype=torch.bfloat16)
    for u, g in ((store[..., :64], store[..., 64:128]), (store[..., 3:67], store[..., 100:164]),
                 (store[:, ::2, :64], store[:, 1::2, 64:128][:, [0, 1, 1]]), (store[..., ::4], store[..., 1::4]),
                 (store[:, :1, :64].expand(-1, 5, -1), store[..., 64:128])):
        want = gated.gated_forward(u.contiguous(), g.contiguous())
        assert torch.equal(gated.gated_forward(u, g), want)
        back, plain = gated.gated_backward(u, u, g), gated.gated_backward(u.contiguous(), u.contiguous(), g.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(back, plain))
    fused = store[..., 5:133]
    want = gated.gated_forward(fused.contiguous())
    assert torch.equal(gated.gated_forward(fused), want)
    assert torch.equal(gated.gated_backward(want, fused), gated.gated_backward(want, fused.contiguous()))
    assert gated.gated_forward(store[:0]).shape == (0, 5, 200)
    out, kept, none = gated.gated_forward(store[:0], keep=True)
    assert none is None and kept.shape == (0, 5, 2, 200) and gated.gated_backward(out, kept).shape == (0, 5, 400)


def test_infinities_and_nan() -> None:
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[inf, -inf, nan, 1.0]], device=DEV)
    u = torch.tensor([[inf, -inf, 2.0]], device=DEV)
    out = gated.gated_forward(torch.ones(1, 4, device=DEV), g)
    exact = _value(torch.ones(1, 4).double(), g.cpu().double(), "situ")
    assert torch.equal(torch.isnan(out).cpu(), torch.isnan(exact)) and out[0, 1] == 0 or out[0, 1] == -0.0
    assert torch.allclose(out.cpu().double()[0, [0, 3]], exact[0, [0, 3]], rtol=1e-6)
    capped = gated.gated_forward(u, torch.full_like(u, 50.0))
    assert torch.allclose(capped.cpu().double(), _value(u.cpu().double(), torch.full((1, 3), 50.0).double(), "situ"), rtol=1e-6)


def test_autograd_matches_differences_and_the_model() -> None:
    both = (2 * _randn(3, 7, 48)).requires_grad_()
    grad = _randn(3, 7, 24, seed=4)
    for kind in gated.KINDS:
        (got,) = torch.autograd.grad(gated.gated(both, kind=kind), both, grad)
        way = _randn(3, 7, 48, seed=5).double()

        def value(t):
            u, g = t.chunk(2, -1)
            return (_value(u, g, kind) * grad.double()).sum()

        wide = both.detach().double()
        slope = (value(wide + 1e-5 * way) - value(wide - 1e-5 * way)) / 2e-5
        # differences are off by 1e-10 times a third derivative of order one, the gradients by 2^-19 of their terms
        assert abs(float((got.double() * way).sum() - slope)) <= 1e-5 * float((got.double() * way).abs().sum())
    up, gate = both.detach().chunk(2, -1)
    # both are fp32 roundings of the same value
    assert torch.allclose(gated.gated_forward(up, gate), dit.situ(up, gate), rtol=2.0**-18, atol=1e-7)


def test_autograd_keeps_8_bits() -> None:
    both = _randn(12, 128, dtype=torch.bfloat16).requires_grad_()
    apart = [t.detach().requires_grad_() for t in both.detach().chunk(2, -1)]
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.dtype), t)[1], lambda t: t):
        out, other = gated.gated(both, keep=True), gated.gated(*apart, keep=True)
    assert saved == [torch.int8, torch.uint8] * 3 and torch.equal(out, other)
    grad = _randn(12, 64, dtype=torch.bfloat16, seed=2)
    (fused,) = torch.autograd.grad(out, both, grad)
    _, kept, _ = gated.gated_forward(both.detach(), keep=True)
    assert torch.equal(fused, gated.gated_backward(grad, kept))
    assert torch.equal(fused, torch.cat(torch.autograd.grad(other, apart, grad), -1))
    with torch.no_grad():
        assert not gated.gated(both, keep=True).requires_grad
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(gated.gated(both).sum(), both, create_graph=True)


def test_refusals() -> None:
    x = _randn(4, 40)
    for bad in ((x[:, :39], None), (x, x[:3]), (x, x.half())):
        with pytest.raises(ValueError):
            gated.gated_forward(*bad)
    with pytest.raises(ValueError):
        gated.gated_forward(x, kind="gelu")
    with pytest.raises(TypeError):
        gated.gated_forward(x.double())
    with pytest.raises(RuntimeError):
        gated.gated_forward(x.requires_grad_())
    x = x.detach()
    out, kept, _ = gated.gated_forward(x, keep=True)
    for bad in ((out[:3], kept), (out, kept, kept), (out.half(), kept), (out, x, x), (out, x[:, :38])):
        with pytest.raises(ValueError):
            gated.gated_backward(*bad)
    with pytest.raises(ValueError):
        gated.gated_backward(out, Kept8(kept.values.flatten(1), kept.exponents.flatten(1), 64, torch.float32))
