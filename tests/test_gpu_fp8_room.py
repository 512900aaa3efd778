"""Every buffer that the 8-bit floating-point and rotary kernels write, or read, at its exact size between guard bytes:
the guards keep their bits, and the results are those of the public calls."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_offload import _native, fp8_kernels as fp8, rotary

from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
GUARD, FILL = 4096, 0xA5
CODES = _native.DTYPE_CODES


class _Room:
    """Buffers of exact sizes in one allocation, 256-byte aligned, at least ``GUARD`` bytes of ``FILL`` between them.
    A read past a buffer finds the fill (a NaN or a large number in every type), a write leaves a mark."""

    def __init__(self, nbytes: int):
        self.bytes = torch.full((nbytes,), FILL, dtype=torch.uint8, device=DEV)
        self.base = -self.bytes.data_ptr() % 256
        self.at, self.taken = self.base + GUARD, []

    def empty(self, *shape, dtype) -> torch.Tensor:
        size = torch.empty((), dtype=dtype).element_size()
        nbytes = size * torch.Size(shape).numel()
        at = self.at
        self.at = (at + nbytes + GUARD - self.base + 255) // 256 * 256 + self.base
        assert self.at <= self.bytes.numel()
        self.taken.append((at, at + nbytes))
        return self.bytes[at : at + nbytes].view(dtype).view(shape)

    def copy(self, tensor: torch.Tensor) -> torch.Tensor:
        to = self.empty(*tensor.shape, dtype=tensor.dtype)
        to.view(torch.uint8).copy_(tensor.contiguous().view(torch.uint8))
        return to

    def check(self) -> None:
        keep = torch.ones(self.bytes.numel(), dtype=torch.bool, device=DEV)
        for start, end in self.taken:
            keep[start:end] = False
        marks = (keep & (self.bytes != FILL)).nonzero().flatten()
        assert not marks.numel(), [int(m) for m in marks[:8]]


def _randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _call(name, *args):
    args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    _native.check(name, getattr(_native.load(), name)(*args, _stream()))


def _same(got, want):
    assert got.shape == want.shape and got.dtype == want.dtype
    assert torch.equal(got.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


# one token up; sizes that end inside a group, a tile, a wave's share and a step
SHAPES = [(1, 16, 16), (1, 3072, 512), (3, 128, 128), (16, 1040, 272), (17, 512, 3136), (33, 144, 400), (65, 1152, 144),
          (130, 272, 1040), (300, 1552, 528), (515, 912, 1296), (1100, 256, 2064), (2050, 1296, 784)]


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("rows,cols", [(r, i) for r, i, _ in SHAPES] + [(127, 4128), (129, 48)])
def test_quantizers_and_read_back_stay_in_their_buffers(rows, cols, dtype) -> None:
    groups, pitch, padded = -(-cols // 128), -(-rows // 16) * 16, -(-rows // 128) * 128
    room = _Room(24 * rows * cols + 4 * cols * padded + 64 * (rows + cols) * groups + (1 << 20))
    x = room.copy(_randn(rows, cols, dtype=dtype))
    want, wanted = fp8.fp8_quantize_both(x)
    for ways in ((1, 0), (0, 1), (1, 1)):
        rv, rs = room.empty(rows, cols, dtype=fp8.E4M3), room.empty(groups, pitch, dtype=torch.uint8)
        cv, cs = room.empty(cols, padded, dtype=fp8.E4M3), room.empty(padded // 128, cols, dtype=torch.uint8)
        _call("mo_fp8_quantize", x, CODES[dtype], rows, cols, cols, *((rv, rs) if ways[0] else (0, 0)),
              *((cv, cs) if ways[1] else (0, 0)))
        room.check()
        for on, values, scales, given, count in ((ways[0], rv, rs, want, rows), (ways[1], cv, cs, wanted, cols)):
            if on:
                _same(values, given[0])
                _same(scales[:, :count].t(), given[1].view(torch.uint8))
            else:
                assert (values.view(torch.uint8) == FILL).all() and (scales == FILL).all()
        if ways[0]:
            assert (rs[:, rows:] == FILL).all()  # the rows that round up to 16 are not written
    wv = room.empty(rows, cols, dtype=fp8.E4M3)
    ws = room.empty(-(-rows // 128), groups, dtype=torch.uint8)
    _call("mo_fp8_quantize_weight", x, CODES[dtype], rows, cols, cols, wv, ws)
    room.check()
    for got, need in zip((wv, ws.view(fp8.E8M0)), fp8.fp8_quantize_weight(x)):
        _same(got, need)
    for width in {cols, cols - 1, cols - 11}:
        out = room.empty(rows, width, dtype=dtype)
        _call("mo_fp8_decode", wv, cols, ws, 0, groups, 1, 128, out, CODES[dtype], rows, width)
        room.check()
        _same(out, fp8.fp8_decode(wv, ws.view(fp8.E8M0), dtype=dtype, cols=width))


@pytest.mark.parametrize("out_dtype", list(CODES))
@pytest.mark.parametrize("floats", [False, True])
@pytest.mark.parametrize("rows,in_features,out_features", SHAPES)
def test_products_stay_in_their_buffers(rows, in_features, out_features, floats, out_dtype) -> None:
    lib, code = _native.load(), CODES[out_dtype]
    weight, scale = fp8.fp8_quantize_weight(0.02 * _randn(out_features, in_features))
    scale = scale.float() * 1.37 if floats else scale
    kind = int(floats)
    tokens, gradient = _randn(rows, in_features, dtype=torch.bfloat16), _randn(rows, out_features, dtype=torch.bfloat16)
    bias = _randn(out_features)
    spaces = {}
    for op in (0, 1, 2):
        for quantized in (0, 1):
            spaces[op, quantized] = lib.mo_fp8_workspace_bytes(op, rows, in_features, out_features, quantized, kind, code)
    size = 4 * (rows * (in_features + out_features) * 2 + in_features * out_features)
    room = _Room(2 * sum(spaces.values()) + 4 * size + (4 << 20))
    w, s, x, dy, b = (room.copy(t) for t in (weight, scale, tokens, gradient, bias))
    outs = [room.empty(*shape, dtype=out_dtype) for shape in ((rows, out_features), (rows, in_features),
                                                              (out_features, in_features))]

    def space(op, quantized):
        nbytes = spaces[op, quantized]
        return (room.empty(nbytes, dtype=torch.uint8), nbytes) if nbytes else (0, 0)

    want = fp8.fp8_linear_forward(tokens, weight, scale, bias, dtype=out_dtype)
    back = fp8.fp8_linear_backward(gradient, weight, scale, dtype=out_dtype)
    grad = fp8.fp8_weight_gradient(gradient, tokens, dtype=out_dtype)
    _call("mo_fp8_linear_forward", x, 0, 1, rows, in_features, in_features, w, s, kind, out_features, b, outs[0],
          code | _native.MO_FP8_BIAS_F32, *space(0, 0))
    _call("mo_fp8_linear_backward", dy, 0, 1, rows, in_features, out_features, out_features, w, s, kind, outs[1], code,
          *space(1, 0))
    _call("mo_fp8_weight_gradient", dy, 0, 1, out_features, x, 0, 1, in_features, rows, in_features, out_features, outs[2],
          code, *space(2, 0))
    room.check()
    for got, need in zip(outs, (want, back, grad)):
        _same(got, need)
        got.view(torch.uint8).fill_(FILL)

    def pair(values, scales):  # the scales' whole pitch, as the quantizers lay them
        pitch = -(-scales.shape[0] // 16) * 16
        laid = room.empty(scales.shape[1], pitch, dtype=torch.uint8)
        laid[:, : scales.shape[0]].copy_(scales.view(torch.uint8).t())
        return room.copy(values), laid

    xr, dr = pair(*fp8.fp8_quantize_rows(tokens)), pair(*fp8.fp8_quantize_rows(gradient))
    xc, dc = pair(*fp8.fp8_quantize_columns(tokens)), pair(*fp8.fp8_quantize_columns(gradient))
    _call("mo_fp8_linear_forward", *xr, 0, rows, in_features, 0, w, s, kind, out_features, b, outs[0],
          code | _native.MO_FP8_BIAS_F32, *space(0, 1))
    _call("mo_fp8_linear_backward", *dr, 0, rows, in_features, out_features, 0, w, s, kind, outs[1], code, *space(1, 1))
    _call("mo_fp8_weight_gradient", *dc, 0, 0, *xc, 0, 0, rows, in_features, out_features, outs[2], code, *space(2, 1))
    room.check()
    for got, need in zip(outs, (want, back, grad)):
        _same(got, need)


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("batch,tokens,heads,kv,head,part", [
    (1, 1, 1, 1, 2, 2), (2, 3, 5, 1, 6, 2), (3, 5, 2, 4, 10, 6), (1, 33, 4, 2, 64, 64), (2, 17, 8, 2, 80, 40),
    (1, 9, 2, 2, 256, 250), (1, 5, 3, 1, 512, 512), (1, 6, 2, 1, 510, 254), (2, 1100, 12, 4, 128, 96)])
def test_rotary_stays_in_its_buffers(batch, tokens, heads, kv, head, part, layout, dtype) -> None:
    lib = _native.load()
    room = _Room(64 * batch * tokens * (heads + kv) * head + (24 << 20))
    sides = [room.copy(_randn(batch, tokens, n, head, dtype=dtype, seed=i)) for i, n in enumerate((heads, kv))]
    grads = [room.copy(_randn(batch, tokens, n, head, dtype=dtype, seed=i + 5)) for i, n in enumerate((heads, kv))]
    weights = [room.copy(1 + 0.1 * _randn(head, seed=i)) for i in (1, 2)]
    table = room.copy(_randn(batch, tokens, part, seed=3))
    outs = [room.empty(*t.shape, dtype=dtype) for t in sides]
    weight_grads = [room.empty(head, dtype=torch.float32) for _ in weights]
    call = _native.MoRotaryCall()
    call.table, call.table_batch, call.table_dtype, call.weight_dtype = table.data_ptr(), tokens * part, 2, 2
    call.dtype, call.batch, call.tokens, call.head_dim, call.rotary_dim = CODES[dtype], batch, tokens, head, part
    call.interleaved, call.eps = layout == "interleaved", 1e-6
    for side, x, grad, out, weight, weight_grad in zip(call.side, sides, grads, outs, weights, weight_grads):
        side.x, side.grad, side.out, side.heads = x.data_ptr(), grad.data_ptr(), out.data_ptr(), x.shape[2]
        side.weight, side.weight_grad = weight.data_ptr(), weight_grad.data_ptr()
        side.x_batch, side.x_token, side.x_head = x.stride()[:3]
        side.grad_batch, side.grad_token, side.grad_head = grad.stride()[:3]
    how = {"layout": layout, "q_weight": weights[0], "k_weight": weights[1]}
    _native.check("mo_rotary_forward", lib.mo_rotary_forward(ctypes.byref(call), _stream()))
    room.check()
    for got, want in zip(outs, rotary.rotary_forward(*sides, table, **how)):
        _same(got, want)
    nbytes = lib.mo_rotary_workspace_bytes(ctypes.byref(call))
    space = room.empty(nbytes, dtype=torch.uint8)
    _native.check("mo_rotary_backward", lib.mo_rotary_backward(ctypes.byref(call), space.data_ptr(), nbytes, _stream()))
    room.check()
    for got, want in zip((*outs, *weight_grads), rotary.rotary_backward(*grads, table, *sides, **how)):
        _same(got, want)


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("rows,axes,bands", [(1, 1, 1), (77, 4, 16), (333, 3, 5), (1000, 1, 64)])
def test_the_table_stays_in_its_buffer(rows, axes, bands, dtype) -> None:
    room = _Room(64 * rows * axes * bands + (1 << 20))
    where, rate = room.copy(_randn(rows, axes)), room.copy(_randn(bands))
    out = room.empty(rows, 2 * axes * bands, dtype=dtype)
    _call("mo_rotary_table", where, rate, out, CODES[dtype], rows, axes, bands, 1.5)
    room.check()
    _same(out, rotary.rotary_table(where, rate, amplitude=1.5, dtype=dtype))
