"""Activations in 8 bits on the GPU, bit for bit with the rule in 64 bits: odd sizes, strides, values at the ends of
their types, infinities and NaN; and checkpointed blocks whose input is kept so."""

from __future__ import annotations

import pytest
import torch

from moss_offload import dit
from moss_offload.kept8 import Kept8, checkpoint_kept8, keep8

from gpu_util import requires_gpu
import kept8_model

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _same(kept: Kept8, x: torch.Tensor) -> None:
    values, exponents = kept8_model.keep(x)
    assert kept.shape == x.shape and kept.dtype == x.dtype
    assert torch.equal(kept.values, values) and torch.equal(kept.exponents, exponents)
    back = kept.restore()
    assert back.shape == x.shape and back.dtype == x.dtype
    # q has seven bits, so it is exact in every type
    assert torch.equal(back.double().nan_to_num(-1.0), kept8_model.read(values, exponents, x.shape[-1]).nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (31,), (1, 1), (3, 32), (5, 33), (2, 3, 7), (17, 64), (129, 100), (4, 5, 96), (64, 1001)])
def test_sizes(shape, dtype) -> None:
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = (torch.randn(*shape, device=DEV, generator=g) * torch.exp(3 * torch.randn(*shape, device=DEV, generator=g))).to(dtype)
    _same(keep8(x), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_peak_of_a_16_bit_type_and_its_half_steps(dtype) -> None:
    """Each 16-bit pattern as a group's largest, beside values that fall on halves of its steps."""

    bits = torch.arange(1 << 16, device=DEV, dtype=torch.int32).to(torch.int16)
    peak = bits.view(dtype) if dtype != torch.float32 else (bits.to(torch.int32) << 16).view(torch.float32)
    part = torch.arange(32, device=DEV, dtype=torch.float64)
    wide = torch.where(torch.isfinite(peak), peak.double(), torch.zeros_like(peak, dtype=torch.float64))
    x = (wide[:, None] * (1 - part / 64)).to(dtype)
    x[:, 0] = peak
    x[:, 5] = -x[:, 5]
    _same(keep8(x), x)


def test_the_ends_of_the_types() -> None:
    for dtype in DTYPES:
        info = torch.finfo(dtype)
        x = torch.zeros(8, 64, device=DEV, dtype=dtype)
        x[0, 3], x[1, 40], x[2, 0], x[3, 63] = info.max, info.min, info.tiny, info.smallest_normal / 4
        x[4, 7], x[5, 33], x[6, 1] = float("inf"), float("-inf"), float("nan")
        x[7] = -0.0
        x[4:7, 10] = 3.0
        kept = keep8(x)
        _same(kept, x)
        back = kept.restore()
        assert torch.isfinite(back[:4]).all() and torch.isnan(back[4, :32]).all() and back[4, 32:].eq(0).all()
        assert torch.isnan(back[5, 32:]).all() and torch.isnan(back[6, :32]).all()


def test_views_and_places() -> None:
    g = torch.Generator(device="cuda").manual_seed(1)
    store = torch.randn(40, 400, device=DEV, generator=g).bfloat16()
    for x in (store[:, 3:200], store[::3, 8:72], store.t(), store[:, ::2], store[5, 7:77], store[:0], store[None, :, :33],
              store[:1].expand(6, -1)):
        _same(keep8(x), x)


def test_another_type_on_the_way_back() -> None:
    x = torch.randn(9, 70, device=DEV)
    exact = kept8_model.read_back(x)
    kept = keep8(x)
    for dtype in DTYPES:
        assert torch.equal(kept.restore(dtype), exact.to(dtype))


def test_off_by_half_a_step_at_most() -> None:
    x = torch.randn(300, 320, device=DEV)
    peak = x.unflatten(1, (10, 32)).abs().amax(-1, keepdim=True)
    # 127 steps reach the peak and 127 of the half steps do not: a step is at most peak * 2 / 127, half of it the error
    off = (keep8(x).restore() - x).unflatten(1, (10, 32)).abs()
    assert (off <= peak / 127 * 1.000001).all()


def test_offsets_past_32_bits() -> None:
    rows, cols = 70_000, 65_536  # 4.6e9 values
    x = torch.zeros(1, cols, device=DEV, dtype=torch.bfloat16).expand(rows, cols)
    x = x.clone()
    last = torch.randn(3, cols, device=DEV).bfloat16()
    x[-3:] = last
    kept = keep8(x)
    values, exponents = kept8_model.keep(last)
    assert torch.equal(kept.values[-3:], values) and torch.equal(kept.exponents[-3:], exponents)
    assert not kept.values[:-3].any()
    del x
    back = kept.restore()
    assert torch.equal(back[-3:].double(), kept8_model.read_back(last)) and not back[:-3].any()


# ---- checkpoints ------------------------------------------------------------------------------------------


def _block():
    torch.manual_seed(3)
    block = dit.Block(64, 128, 4).to(DEV)
    dit.init_weights(block, std=0.1)
    tokens = torch.randn(1, 20, 64, device=DEV, requires_grad=True)
    rope = torch.randn(1, 20, 16, device=DEV)
    modulation = torch.randn(1, 6, 64, device=DEV, requires_grad=True)
    return block, tokens, rope, modulation


def test_a_checkpoint_gives_the_exact_result_and_the_kept_inputs_gradients() -> None:
    block, tokens, rope, modulation = _block()
    out = checkpoint_kept8(block, tokens, rope, modulation, None, None)
    assert torch.equal(out, block(tokens, rope, modulation))
    grad = torch.randn_like(out)
    out.backward(grad)
    got = [tokens.grad, modulation.grad, *(p.grad for p in block.parameters())]
    kept = kept8_model.read_back(tokens.detach()).float().requires_grad_()
    want = torch.autograd.grad(block(kept, rope, modulation), [kept, modulation, *block.parameters()], grad)
    # the same kernels on the same bits; library reductions may sum in another order
    for g, w in zip(got, want):
        assert torch.allclose(g, w, rtol=1e-4, atol=1e-4 * float(w.abs().max()))


def test_a_checkpoint_replays_random_numbers_and_autocast() -> None:
    layer = torch.nn.Linear(32, 32).to(DEV)
    seen = []

    def run(tokens):
        out = torch.nn.functional.dropout(layer(tokens), 0.5)
        seen.append((out.dtype, (out == 0).clone()))
        return out

    x = torch.randn(40, 32, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = checkpoint_kept8(run, x)
    state = torch.cuda.get_rng_state()
    out.sum().backward()
    assert torch.equal(torch.cuda.get_rng_state(), state)
    assert seen[0][0] == seen[1][0] == torch.bfloat16 and torch.equal(seen[0][1], seen[1][1])


def test_what_a_checkpoint_refuses() -> None:
    block, tokens, rope, modulation = _block()
    with pytest.raises(RuntimeError, match="requires grad"):
        checkpoint_kept8(block, tokens.detach(), rope, modulation.detach())
    with torch.no_grad():
        assert not checkpoint_kept8(block, tokens, rope, modulation).requires_grad
    out = checkpoint_kept8(block, tokens, rope, modulation)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out.sum(), tokens, create_graph=True)
