"""The workspace of an adapters' backward pass goes by the adapters that its requests can have, not by the pool they are from."""

from __future__ import annotations

import ctypes

import pytest

from moss_offload import _native

P = 1 << 20  # an address that nothing reads


@pytest.mark.parametrize("requests", [1, 3])
def test_room_for_a_pool(requests) -> None:
    def needed(adapters, **gradients):
        call = _native.MoAdaptersCall()
        for name in ("x", "a", "b", "hidden", "grad", "index", "cu"):
            setattr(call, name, P)
        call.rows, call.in_features, call.out_features, call.rank, call.dtype = 60, 256, 128, 16, 1
        call.x_stride, call.grad_stride, call.requests, call.adapters, call.factor = 256, 128, requests, adapters, 1.0
        for name in gradients:
            setattr(call, name, P)
        nbytes = _native.load().mo_adapters_workspace_bytes(ctypes.byref(call), 1)
        assert nbytes
        return nbytes

    assert needed(requests, dx=1) == needed(requests + 1, dx=1) == needed(20000, dx=1)
    assert needed(requests, dx=1, da=1) == needed(20000, dx=1, da=1)
    if requests > 1:
        assert needed(1, dx=1) < needed(requests, dx=1)
