"""The rotary calls through their C ABI on the GPU: tables whose batch entries lie any distance apart."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_offload import _native, rotary

from gpu_util import requires_gpu
from test_gpu_rotary import _close, _exact

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("spare", [0, 1, 2, 4, 8, 13])
@pytest.mark.parametrize("table_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
def test_tables_any_distance_apart(layout, table_dtype, spare) -> None:
    lib = _native.load()
    batch, tokens, heads, head, part = 3, 21, 4, 32, 16
    g = torch.Generator(device="cuda").manual_seed(spare)
    x, grad = (torch.randn(batch, tokens, heads, head, device=DEV, generator=g).bfloat16() for _ in range(2))
    pitch = tokens * part + spare
    room = torch.full((batch * pitch,), float("nan"), device=DEV).to(table_dtype)
    table = room.view(batch, pitch)[:, : tokens * part].unflatten(1, (tokens, part))
    table.copy_(torch.randn(batch, tokens, part, device=DEV, generator=g).to(table_dtype))
    out = torch.empty_like(x)
    call = _native.MoRotaryCall()
    call.table, call.table_batch, call.table_dtype = room.data_ptr(), pitch, _native.DTYPE_CODES[table_dtype]
    call.dtype, call.batch, call.tokens, call.head_dim, call.rotary_dim = 1, batch, tokens, head, part
    call.interleaved = layout == "interleaved"
    side = call.side[0]
    side.heads, side.out = heads, out.data_ptr()
    side.x, side.x_batch, side.x_token, side.x_head = x.data_ptr(), *x.stride()[:3]
    stream = torch.cuda.current_stream().cuda_stream
    _native.check("mo_rotary_forward", lib.mo_rotary_forward(ctypes.byref(call), stream))
    # two products and a sum in fp32, then the rounding to bfloat16
    _close(out, *_exact(x, table, layout, None), torch.bfloat16, 3)
    side.x, side.grad, side.grad_batch, side.grad_token, side.grad_head = 0, grad.data_ptr(), *grad.stride()[:3]
    _native.check("mo_rotary_backward", lib.mo_rotary_backward(ctypes.byref(call), 0, 0, stream))
    back = torch.cat((-table[..., : part // 2], table[..., part // 2 :]), -1)  # the turn by the opposite angle
    _close(out, *_exact(grad, back, layout, None), torch.bfloat16, 3)
