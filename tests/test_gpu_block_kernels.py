"""Norms, gated activations, adapters and 8-bit activations together, as a block uses them: chains under autograd, blocks
and models against 64 bits, the activation offload, graphs, streams, threads, and buffers at their exact sizes."""

from __future__ import annotations

import copy
import threading

import pytest
import torch

import moss_offload
from moss_offload import adapters, dit, gated, norms
from moss_offload.kept8 import checkpoint_kept8, keep8

from gpu_util import assert_bitwise, requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


def _randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


class Chain:
    """A feed-forward of a packed batch: norm and modulation, a projection with an adapter for each sample, the gated
    activation, a projection back."""

    def __init__(self, dtype=torch.bfloat16, rows=90, dim=96, ffn=160, rank=8):
        self.x, self.grad = _randn(rows, dim, dtype=dtype), _randn(rows, dim, dtype=dtype, seed=1)
        self.weight = 1 + 0.1 * _randn(dim, seed=2)
        self.scale, self.shift = (0.2 * _randn(3, dim, dtype=dtype, seed=s) for s in (3, 4))
        self.up, self.down = 0.1 * _randn(2 * ffn, dim, dtype=dtype, seed=5), 0.1 * _randn(dim, ffn, dtype=dtype, seed=6)
        self.a1, self.b1 = 0.1 * _randn(2, rank, dim, dtype=dtype, seed=7), 0.1 * _randn(2, 2 * ffn, rank, dtype=dtype, seed=8)
        self.a2, self.b2 = 0.1 * _randn(2, rank, ffn, dtype=dtype, seed=9), 0.1 * _randn(2, dim, rank, dtype=dtype, seed=10)
        self.cu = torch.tensor([0, 17, 60, rows], device=DEV)
        self.index = torch.tensor([1, 0, 1], device=DEV)

    def leaves(self):
        return [self.x, self.weight, self.scale, self.shift, self.a1, self.b1, self.a2, self.b2]

    def autograd(self, keep):
        x, weight, scale, shift, a1, b1, a2, b2 = leaves = [t.detach().clone().requires_grad_() for t in self.leaves()]
        how = {"cu_seqlens": self.cu, "index": self.index, "keep": keep}
        hidden = norms.norm(x, weight, scale=scale, shift=shift, cu_seqlens=self.cu, keep=keep)
        both = adapters.adapters(hidden, hidden @ self.up.t(), a1, b1, 0.5, **how)
        active = gated.gated(both, keep=keep)
        out = adapters.adapters(active, active @ self.down.t(), a2, b2, 0.5, **how)
        out.backward(self.grad)
        return out.detach(), [t.grad for t in leaves]

    def calls(self, keep):
        norm = {"scale": self.scale, "shift": self.shift, "cu_seqlens": self.cu}
        how = {"cu_seqlens": self.cu, "index": self.index}
        hidden, stats, x = norms.norm_forward(self.x, self.weight, stats=True, keep=keep, **norm)
        both, h1 = adapters.adapters_forward(hidden, hidden @ self.up.t(), self.a1, self.b1, 0.5, hidden=True, **how)
        active, *parts = gated.gated_forward(both, keep=True) if keep else (gated.gated_forward(both), both, None)
        out, h2 = adapters.adapters_forward(active, active @ self.down.t(), self.a2, self.b2, 0.5, hidden=True, **how)
        kept = keep8 if keep else (lambda t: t)
        # autograd adds the two ways into a product's input in its type
        d_active, a2, b2 = adapters.adapters_backward(self.grad, kept(active), h2, self.a2, self.b2, 0.5, **how)
        d_both = gated.gated_backward(d_active + self.grad @ self.down, *parts)
        d_hidden, a1, b1 = adapters.adapters_backward(d_both, kept(hidden), h1, self.a1, self.b1, 0.5, **how)
        back = norms.norm_backward(d_hidden + d_both @ self.up, x if keep else self.x, stats, self.weight, **norm)
        return out, [back.x, back.weight, back.scale, back.shift, a1, b1, a2, b2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("keep", [False, True])
def test_a_chain_under_autograd_is_the_chain_of_calls(keep, dtype) -> None:
    chain = Chain(dtype)
    out, grads = chain.autograd(keep)
    want, wanted = chain.calls(keep)
    assert torch.equal(out, want)
    for g, w in zip(grads, wanted):
        assert torch.equal(g, w)


def _step(block, tokens, rope, modulation, cu, grad):
    tokens, modulation = tokens.detach().clone().requires_grad_(), modulation.detach().clone().requires_grad_()
    block.zero_grad(set_to_none=True)
    out = block(tokens, rope, modulation, cu)
    out.backward(grad)
    return [out.detach(), tokens.grad, modulation.grad, *(p.grad for p in block.parameters() if p.requires_grad)]


def _block(packed, lora=True):
    torch.manual_seed(5)
    model = dit.MOSSImageTransformer(dim=64, ffn_dim=96, num_heads=4, num_layers=1, text_dim=32, freq_dim=16, latent_channels=8)
    dit.init_weights(model, std=0.08)
    if lora:
        dit.inject_lora(model, rank=8, alpha=4.0)
    block = model.layers[0].to(DEV)
    samples = 3 if packed else 1
    cu = torch.tensor([0, 9, 30, 44], device=DEV) if packed else None
    inputs = _randn(1, 44, 64), _randn(1, 44, 16, seed=1), 0.3 * _randn(samples, 6, 64, seed=2), cu, _randn(1, 44, 64, seed=3)
    return block, inputs


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lora", [False, True])
def test_a_block_is_as_near_to_64_bits_as_the_composed_one(lora, packed) -> None:
    block, inputs = _block(packed, lora)
    wide = copy.deepcopy(block).double()
    exact = _step(wide, *(t.double() if t is not None and t.is_floating_point() else t for t in inputs))
    plain = _step(block, *inputs)
    assert dit.configure_kernels(block, "hip") == (1 + 6 if lora else 1)
    fused = _step(block, *inputs)
    for e, p, f in zip(exact, plain, fused):
        size = float(e.abs().max())
        # both are fp32 throughout; 2^-20 of the largest stands for sums of up to 100 terms in another order
        assert float((f - e).abs().max()) <= 2 * float((p - e).abs().max()) + 2.0**-20 * size


def test_a_block_in_8_bits_gives_the_same_output_and_near_gradients() -> None:
    block, inputs = _block(True)
    dit.configure_kernels(block, "hip")
    whole = _step(block, *inputs)
    dit.configure_kernels(block, "hip", keep8=True)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.dtype), t)[1], lambda t: t):
        kept = _step(block, *inputs)
    assert torch.equal(whole[0], kept[0]) and torch.int8 in saved
    for w, k in zip(whole[1:], kept[1:]):
        # a value is off by 2^-8 of its group's largest (half a step of 2^-7) at most, some thousandths of the norm on the whole;
        # through four such tensors the gradients stay within a few hundredths
        assert float((w - k).norm()) <= 0.04 * float(w.norm())
    # the last d b is a product of the output's gradient and the forward pass's h, neither of which went through 8 bits
    assert not torch.equal(whole[1], kept[1])
    for bad in (("fused", False), ("composed", True)):
        with pytest.raises(ValueError):
            dit.configure_kernels(block, bad[0], keep8=bad[1])


def _model(**how):
    torch.manual_seed(0)
    model = dit.MOSSImageTransformer(dim=64, ffn_dim=128, num_heads=4, num_layers=3, text_dim=32, freq_dim=16, latent_channels=8, **how)
    dit.init_weights(model)
    dit.inject_lora(model, rank=4, alpha=4.0)
    model = model.to(DEV).to(torch.bfloat16).train()
    dit.configure_kernels(model, "hip", keep8=True)
    return model


def _train(model, packed, offload):
    model.activation_offload = offload
    model.zero_grad(set_to_none=True)
    if packed:
        latents, context = [_randn(8, 4, 4), _randn(8, 2, 6, seed=1)], [_randn(6, 32, seed=2), _randn(9, 32, seed=3)]
        outs = model.forward_packed([t.bfloat16() for t in latents], torch.tensor([500.0, 100.0], device=DEV),
                                    [t.bfloat16() for t in context])
        loss = sum(o.float().square().mean() for o in outs)
    else:
        loss = model(_randn(1, 8, 4, 4).bfloat16(), torch.tensor([500.0], device=DEV), _randn(1, 6, 32, seed=2).bfloat16()).float().square().mean()
    loss.backward()
    return [loss.detach(), *(p.grad.detach().clone() for p in model.parameters() if p.requires_grad)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("how", [{}, {"gradient_checkpointing": True}, {"gradient_checkpointing": True, "checkpoint_keep8": True}])
def test_a_model_under_the_activation_offload_bit_for_bit(how, packed) -> None:
    model = _model(**how)
    resident = _train(model, packed, False)
    offloaded = _train(model, packed, True)
    torch.cuda.synchronize()
    assert moss_offload.get_engine(DEV).stats()["bytes_packed"] > 0
    for r, o in zip(resident, offloaded):
        assert_bitwise(o, r)


def test_a_checkpoint_in_8_bits_in_the_model() -> None:
    exact = _train(_model(gradient_checkpointing=True), False, False)
    kept = _train(_model(gradient_checkpointing=True, checkpoint_keep8=True), False, False)
    assert torch.equal(exact[0], kept[0])
    for e, k in zip(exact[1:], kept[1:]):
        assert torch.isfinite(k).all() and float((e - k).norm()) <= 0.2 * float(e.norm()) + 1e-6


# ---- graphs, streams, threads -----------------------------------------------------------------------------


@pytest.mark.parametrize("keep", [False, True])
def test_a_captured_chain_replays_with_new_inputs(keep) -> None:
    chain, other = Chain(rows=300, dim=512, ffn=256), Chain(rows=300, dim=512, ffn=256)
    other.x, other.grad = 2 * _randn(300, 512, dtype=torch.bfloat16, seed=77), _randn(300, 512, dtype=torch.bfloat16, seed=78)
    eager, eager_other = chain.calls(keep), other.calls(keep)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        chain.calls(keep)
    torch.cuda.synchronize()
    first = chain.x.clone(), chain.grad.clone()
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = chain.calls(keep)
        graphs.append((graph, result))
    for turn in range(4):
        for (x, grad), (out, grads) in ((first, eager), ((other.x, other.grad), eager_other)):
            chain.x.copy_(x)
            chain.grad.copy_(grad)
            graph, (got, gots) = graphs[turn % 2]
            graph.replay()
            Chain(rows=40).calls(keep)  # the program's own work in between
            torch.cuda.synchronize()
            assert torch.equal(got, out)
            for g, w in zip(gots, grads):
                assert torch.equal(g, w)


def test_another_stream() -> None:
    chain = Chain()
    want = chain.calls(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = chain.calls(True)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(g, w) for g, w in zip(got[1], want[1]))


def test_two_threads_at_once() -> None:
    chains = [Chain(), Chain(rows=120, dim=128, ffn=96)]
    want = [c.calls(True) for c in chains]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    out, grads = chains[i].calls(True)
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(out, want[i][0]) and all(torch.equal(g, w) for g, w in zip(grads, want[i][1]))
        except BaseException as error:  # noqa: BLE001
            failed.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_a_checkpoint_of_fused_blocks_accumulates_once() -> None:
    block, (tokens, rope, modulation, cu, grad) = _block(False)
    dit.configure_kernels(block, "hip")
    tokens.requires_grad_()
    for _ in range(2):
        checkpoint_kept8(block, tokens, rope, modulation).backward(grad)
    twice = [p.grad.clone() for p in block.parameters() if p.requires_grad]
    block.zero_grad(set_to_none=True)
    checkpoint_kept8(block, tokens, rope, modulation).backward(grad)
    for t, p in zip(twice, (p for p in block.parameters() if p.requires_grad)):
        assert torch.allclose(t, 2 * p.grad, rtol=1e-5, atol=1e-6)


# ---- buffers at their exact sizes ---------------------------------------------------------------------------


class Guarded:
    """Every tensor that is made while this is in force lies between 256 bytes that must stay as they are."""

    GUARD = 256

    def __init__(self, monkeypatch):
        self.rooms, self.empty = [], torch.empty
        monkeypatch.setattr(torch, "empty_like", lambda t, dtype=None, memory_format=None: self.make(t.shape, dtype or t.dtype))
        monkeypatch.setattr(torch.Tensor, "new_empty", lambda t, shape, dtype=None: self.make(shape, dtype or t.dtype))

    def make(self, shape, dtype):
        shape = (shape,) if isinstance(shape, int) else tuple(shape)
        nbytes = torch.Size(shape).numel() * torch.zeros((), dtype=dtype).element_size()
        room = self.empty(2 * self.GUARD + nbytes, dtype=torch.uint8, device=DEV)
        room.fill_(0xA5)
        self.rooms.append((room, nbytes))
        return room[self.GUARD : self.GUARD + nbytes].view(dtype).view(shape)

    def check(self):
        assert self.rooms
        for room, nbytes in self.rooms:
            assert room[: self.GUARD].eq(0xA5).all() and room[self.GUARD + nbytes :].eq(0xA5).all()


def _surrounded(t):
    """``t`` in the middle of infinities, on the same 256-byte grid: what is read past it would show."""

    room = torch.full((t.numel() + 1024,), float("inf"), dtype=t.dtype, device=DEV)
    room[512 : 512 + t.numel()] = t.flatten()
    return room[512 : 512 + t.numel()].view(t.shape)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,dim,ffn,rank", [(1, 8, 8, 8), (70, 33, 7, 5), (33, 520, 136, 24), (130, 1000, 264, 64), (90, 128, 1032, 16)])
def test_buffers_at_their_exact_sizes(rows, dim, ffn, rank, dtype, monkeypatch) -> None:
    chain = Chain(dtype, rows, dim, ffn, rank)
    cuts = sorted((0, rows // 5, rows - rows // 4, rows))
    chain.cu = torch.tensor(cuts, device=DEV)
    want = [chain.calls(keep) for keep in (False, True)]
    for name in ("x", "grad", "weight", "scale", "shift", "a1", "b1", "a2", "b2"):
        setattr(chain, name, _surrounded(getattr(chain, name)))
    guarded = Guarded(monkeypatch)
    got = [chain.calls(keep) for keep in (False, True)]
    torch.cuda.synchronize()
    guarded.check()
    for (out, grads), (plain, plains) in zip(got, want):
        assert torch.equal(out, plain)
        for g, w in zip(grads, plains):
            assert torch.equal(g, w)
