"""Rotary positions on the GPU against 64 bits: both layouts, parts of heads, odd sizes, views, tables by batch
entry, the heads' norm, and the gradients, by the formula and by differences."""

from __future__ import annotations

import math

import pytest
import torch

from moss_offload import dit, rotary

from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ROUNDING = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _table(batch, tokens, rotary_dim, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    angle = 100 * torch.rand(batch, tokens, rotary_dim // 2, device=DEV, generator=g)
    return torch.cat((angle.sin(), angle.cos()), -1).to(dtype)


def _exact(x, table, layout, weight, eps=1e-6):
    """The definition in 64 bits, differentiable; and the same with absolute values, for the bound."""

    x, table = x.double(), table.double().unsqueeze(2)
    half = table.shape[-1] // 2
    sin, cos = table[..., :half], table[..., half:]
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    part = x[..., : 2 * half]
    first, second = (part[..., :half], part[..., half:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    turned = (first * cos - second * sin, second * cos + first * sin)
    size = (first.abs() * cos.abs() + second.abs() * sin.abs(), second.abs() * cos.abs() + first.abs() * sin.abs())
    join = (lambda p: torch.cat(p, -1)) if layout == "half" else (lambda p: torch.stack(p, -1).flatten(-2))
    rest = x[..., 2 * half :]
    return torch.cat((join(turned), rest), -1), torch.cat((join(size), rest.abs()), -1)


def _close(got, exact, size, dtype, steps):
    """``steps`` fp32 roundings of terms no larger than ``size``, then the output's rounding."""

    near = steps * 2.0**-24 * size
    bound = near + ROUNDING[dtype] * (exact.abs() + near) + (2.0**-25 if dtype == torch.float16 else 2.0**-126)
    worst = ((got.double() - exact).abs() / bound).max()
    assert worst <= 1, float(worst)


# batch, tokens, query heads, key heads, head_dim, rotary_dim
SHAPES = [(1, 1, 1, 1, 2, 2), (2, 3, 5, 1, 6, 2), (1, 7, 3, 3, 8, 8), (3, 5, 2, 4, 10, 6), (1, 33, 4, 2, 64, 64),
          (2, 17, 8, 2, 80, 40), (1, 130, 3, 3, 96, 48), (2, 65, 24, 24, 128, 128), (16, 1, 32, 8, 128, 64),
          (1, 9, 2, 2, 256, 250), (1, 5, 3, 1, 512, 512), (1, 6, 2, 1, 510, 254), (1, 600, 7, 7, 128, 96), (2, 1100, 12, 4, 128, 96), (1, 2100, 8, 8, 40, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("batch,tokens,heads,kv,head,part", SHAPES)
def test_forward_and_backward_match_64_bits(batch, tokens, heads, kv, head, part, norm, layout, dtype) -> None:
    q, k = _randn(batch, tokens, heads, head, dtype=dtype), _randn(batch, tokens, kv, head, dtype=dtype, seed=1)
    grads = [_randn(batch, tokens, n, head, dtype=dtype, seed=2) for n in (heads, kv)]
    table = _table(batch, tokens, part)
    weights = [1 + 0.2 * _randn(head, seed=s) for s in (3, 4)] if norm else [None, None]
    how = {"layout": layout, "q_weight": weights[0], "k_weight": weights[1]}
    outs = rotary.rotary_forward(q, k, table, **how)
    back = rotary.rotary_backward(*grads, table, *((q, k) if norm else ()), **how)
    for x, grad, weight, out, dx, dw in zip((q, k), grads, weights, outs, back[:2], back[2:]):
        leaf = x.double().requires_grad_()
        w = weight.double().requires_grad_() if norm else None
        exact, size = _exact(leaf, table, layout, w)
        # the norm: a sum of head_dim squares under a root, two products; the turn: two products and a sum
        steps = (head / 2 + 8 if norm else 0) + 3
        _close(out, exact.detach(), size.detach(), dtype, steps)
        wanted = torch.autograd.grad(exact, [leaf, w] if norm else [leaf], grad.double())
        # the input's gradient: the turned gradient (as large as the larger of its pair), then r (g w - n
        # mean(g w n)), whose two terms are at most r max|w| |g| and r |n| max|w| |g| mean over the head
        g_size = _exact(grad.double(), table, layout, None)[1]
        if not norm:
            _close(dx, wanted[0], g_size, dtype, 3)
            assert dw is None
            continue
        rms = (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
        unit = x.double() / rms
        scaled = g_size * weight.double().abs()
        bound = (scaled + unit.abs() * (scaled * unit.abs()).mean(-1, keepdim=True)) / rms
        _close(dx, wanted[0], bound, dtype, 3 * steps + head)
        rows = batch * tokens * x.shape[2]
        assert dw.dtype == weight.dtype
        _close(dw, wanted[1], (g_size * unit.abs()).sum((0, 1, 2)), torch.float32, steps + rows)


@pytest.mark.parametrize("table_dtype", DTYPES)
@pytest.mark.parametrize("weight_dtype", DTYPES)
def test_types_of_table_and_weights(table_dtype, weight_dtype) -> None:
    q, k = _randn(2, 20, 3, 64, dtype=torch.bfloat16), _randn(2, 20, 3, 64, dtype=torch.bfloat16, seed=1)
    table = _table(2, 20, 64, table_dtype)
    weights = [(1 + 0.2 * _randn(64, seed=s)).to(weight_dtype) for s in (3, 4)]
    outs = rotary.rotary_forward(q, k, table, q_weight=weights[0], k_weight=weights[1])
    for x, weight, out in zip((q, k), weights, outs):
        exact, size = _exact(x, table, "half", weight)
        _close(out, exact, size, torch.bfloat16, 43)
    back = rotary.rotary_backward(q, k, table, q, k, q_weight=weights[0], k_weight=weights[1])
    assert back[2].dtype == back[3].dtype == weight_dtype


@pytest.mark.parametrize("layout", rotary.LAYOUTS)
def test_views_of_a_fused_projection_and_odd_places(layout) -> None:
    """Slices, transposes, steps, expanded heads and rows off the 16-byte grid give what copies of them give."""

    fused = _randn(3, 40, 6 * 64 + 8, dtype=torch.bfloat16)
    q = fused[..., : 2 * 64].unflatten(-1, (2, 64))
    odd = fused[..., 3 : 3 + 2 * 64].unflatten(-1, (2, 64))
    turned = _randn(3, 2, 40, 64, dtype=torch.bfloat16).transpose(1, 2)
    stepped = fused[:, ::2, 128:384].unflatten(-1, (4, 64))[:, :, ::2]
    spread = fused[:, :, None, :64].expand(-1, -1, 5, -1)
    strided = _randn(3, 40, 2, 128, dtype=torch.bfloat16)[..., ::2]
    weight = 1 + 0.1 * _randn(64)
    for x in (q, odd, turned, stepped, spread, strided):
        table = _table(1, x.shape[1], 32)
        for w in (None, weight):
            got = rotary.rotary_forward(x, None, table, layout=layout, q_weight=w)[0]
            want = rotary.rotary_forward(x.contiguous(), None, table, layout=layout, q_weight=w)[0]
            assert got.is_contiguous()
            exact, size = _exact(x, table, layout, w)
            _close(got, exact, size, torch.bfloat16, 43)
            assert torch.allclose(got.float(), want.float(), rtol=2.0**-7, atol=1e-6)
            back = rotary.rotary_backward(x, None, table, x if w is not None else None, layout=layout, q_weight=w)
            copy = x.contiguous()
            again = rotary.rotary_backward(copy, None, table, copy if w is not None else None, layout=layout, q_weight=w)
            assert torch.allclose(back[0].float(), again[0].float(), rtol=2.0**-6, atol=1e-4)


def test_tables_off_the_grid_and_shared_tables() -> None:
    q = _randn(4, 30, 2, 64)
    store = _randn(1 + 4 * 30 * 64)
    table = store[1:].view(4, 30, 64)
    got = rotary.rotary_forward(q, None, table)[0]
    _close(got, *_exact(q, table, "half", None), torch.float32, 3)
    shared = rotary.rotary_forward(q, None, table[:1])[0]
    assert torch.equal(shared, rotary.rotary_forward(q, None, table[:1].expand(4, -1, -1).contiguous())[0])
    assert torch.equal(shared, rotary.rotary_forward(q, None, table[0])[0])


def test_empty_sides() -> None:
    table = _table(1, 6, 8)
    q = _randn(2, 6, 3, 8)
    none = _randn(2, 6, 0, 8)
    weight = torch.ones(8, device=DEV)
    out = rotary.rotary_forward(q, none, table, q_weight=weight, k_weight=weight)
    assert out[1].shape == none.shape and torch.equal(out[0], rotary.rotary_forward(q, None, table, q_weight=weight)[0])
    back = rotary.rotary_backward(q, none, table, q, none, q_weight=weight, k_weight=weight)
    assert back[1].shape == none.shape and not back[3].any()
    assert torch.equal(rotary.rotary_backward(None, q, table)[1], rotary.rotary_backward(q, None, table)[0])
    nothing = rotary.rotary_backward(q[:, :0], None, table[:, :0], q[:, :0], q_weight=weight)
    assert nothing[0].shape == (2, 0, 3, 8) and not nothing[2].any()


def test_values_that_are_not_finite_stay_in_their_head() -> None:
    q = _randn(1, 8, 4, 64)
    clean = rotary.rotary_forward(q, None, _table(1, 8, 64), q_weight=torch.ones(64, device=DEV))[0]
    q[0, 3, 2, 5] = float("nan")
    got = rotary.rotary_forward(q, None, _table(1, 8, 64), q_weight=torch.ones(64, device=DEV))[0]
    assert got[0, 3, 2].isnan().all()
    keep = torch.ones(1, 8, 4, dtype=torch.bool, device=DEV)
    keep[0, 3, 2] = False
    assert torch.equal(got[keep], clean[keep])
    zero = rotary.rotary_forward(torch.zeros_like(q), None, _table(1, 8, 64), q_weight=torch.ones(64, device=DEV))[0]
    assert not zero.any()


@pytest.mark.parametrize("axes,bands,dtype", [(1, 64, torch.float32), (4, 16, torch.float32), (4, 16, torch.bfloat16),
                                              (3, 5, torch.float16)])
def test_table_is_the_models(axes, bands, dtype) -> None:
    """Coordinates up to a million: the angle is the float32 product, its sine and cosine right to two units."""

    rate = 1 / 10000 ** (torch.arange(bands, device=DEV, dtype=torch.float64) / bands)
    coordinates = (torch.randint(-1000, 1_000_000, (2, 50, axes), device=DEV).float() / 2).contiguous()
    table = rotary.rotary_table(coordinates, rate.float(), amplitude=1.25, dtype=dtype)
    phase = (coordinates.unsqueeze(-1) * rate.float()).flatten(-2).double()
    exact = 1.25 * torch.cat((phase.sin(), phase.cos()), -1)
    assert table.shape == (2, 50, 2 * axes * bands) and table.dtype == dtype
    assert ((table.double() - exact).abs() <= 4 * 2.0**-24 * 1.25 + ROUNDING[dtype] * exact.abs() + 2.0**-24).all()
    if axes == 4 and dtype == torch.float32:
        plain = rotary.rotary_table(coordinates[0], rate.float())
        assert torch.allclose(plain, dit.rope_phases(coordinates[0], rate.float())[0], rtol=0, atol=5e-7)


def test_gradients_under_autograd_and_by_differences() -> None:
    q, k = _randn(2, 9, 3, 16).requires_grad_(), _randn(2, 9, 1, 16, seed=1).requires_grad_()
    weights = [(1 + 0.2 * _randn(16, seed=s)).requires_grad_() for s in (3, 4)]
    table = _table(2, 9, 12)
    probes = [_randn(*t.shape, seed=7) for t in (q, k)]
    leaves = [q, k, *weights]

    def loss(q, k, a, b):
        out = rotary.rotary(q, k, table, layout="interleaved", q_weight=a, k_weight=b)
        return sum((o.double() * p.double()).sum() for o, p in zip(out, probes))

    got = torch.autograd.grad(loss(*leaves), leaves)
    step = 2.0**-9
    for which, leaf in enumerate(leaves):
        for index in [(0,) * leaf.ndim, tuple(s - 1 for s in leaf.shape), tuple(s // 2 for s in leaf.shape)]:
            values = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[which][index] += sign * step
                values.append(float(loss(*moved)))
            # a central difference: fp32 outputs round each term by 2^-24, the cube term is step^2
            assert float(got[which][index]) == pytest.approx((values[0] - values[1]) / (2 * step), rel=2e-3, abs=5e-3)
    plain = rotary.rotary(q, k, table)
    grads = torch.autograd.grad([plain[0]], [q], [probes[0]])
    assert torch.equal(grads[0], rotary.rotary_backward(probes[0], None, table)[0])


def test_without_a_norm_the_heads_are_not_kept() -> None:
    q = _randn(1, 5, 2, 16).requires_grad_()
    table = _table(1, 5, 16)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.data_ptr()) or t, lambda t: t):
        rotary.rotary(q, None, table)
    assert saved == [table.data_ptr()]


def test_the_same_call_gives_the_same_bits_from_a_stream_and_a_graph() -> None:
    q, k = _randn(1, 700, 24, 128, dtype=torch.bfloat16), _randn(1, 700, 24, 128, dtype=torch.bfloat16, seed=1)
    table, weight = _table(1, 700, 128), 1 + 0.1 * _randn(128)
    how = {"q_weight": weight, "k_weight": weight}

    def calls():
        return [*rotary.rotary_forward(q, k, table, **how), *rotary.rotary_backward(q, k, table, q, k, **how)]

    want = calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [calls() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for each in got:
        assert all(torch.equal(a, b) for a, b in zip(each, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for seed in range(3):
        q.copy_(_randn(1, 700, 24, 128, dtype=torch.bfloat16, seed=seed + 5))
        want = calls()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("method", rotary.SCALINGS)
def test_scaled_bands_turn_long_positions_as_the_trained_ones(method) -> None:
    bands = (1 / 10000 ** (torch.arange(64, dtype=torch.float64) / 64)).float().to(DEV)
    scaled, amplitude = rotary.scaled_bands(bands, 8.0, method)
    positions = torch.arange(0, 4096, 64, device=DEV, dtype=torch.float32)[:, None]
    long = rotary.rotary_table(positions * 8, scaled, amplitude=amplitude)
    short = rotary.rotary_table(positions, bands)
    assert amplitude == (0.1 * math.log(8) + 1 if method == "yarn" else 1.0)
    last = [63, 127]  # the slowest band is divided by the factor under every method
    assert torch.allclose(long[:, last], amplitude * short[:, last], atol=1e-4)
