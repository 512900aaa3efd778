"""The rotary calls without a device: which lanes a call gets through the C ABI, seen in the size of its partial sums,
and what autograd refuses."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_offload import _native, rotary


def _lanes(**fields) -> int:
    """Lanes a head of 16 fp16 values in a backward call with a norm: its workgroups of 256 lanes leave 16 floats each."""

    call = _native.MoRotaryCall()
    call.table, call.batch, call.tokens, call.head_dim, call.rotary_dim = 4096, 2, 500, 16, 16
    side = call.side[0]
    side.x = side.out = side.grad = side.weight = side.weight_grad = 4096
    side.heads = 16
    for name in ("x", "grad"):
        for i, step in enumerate(("head", "token", "batch")):
            setattr(side, f"{name}_{step}", (16, 256, 500 * 256)[i])
    call.table_batch, call.table_dtype = 500 * 16, 2
    for name, value in fields.items():
        setattr(call if hasattr(call, name) else side, name, value)
    nbytes = _native.load().mo_rotary_workspace_bytes(ctypes.byref(call))
    workgroups = nbytes // 64
    assert nbytes % 64 == 0 and workgroups < 1024
    return round(workgroups * 256 / (2 * 500 * 16))


@pytest.mark.parametrize("table_dtype", [0, 1, 2])
@pytest.mark.parametrize("table_batch,lanes", [(0, 1), (8000, 1), (8008, 1), (8004, 2), (8002, 4), (8001, 8), (1, 8)])
def test_a_tables_batch_stride_is_part_of_its_alignment(table_batch, lanes, table_dtype) -> None:
    """A lane reads its pairs' angles by 16 bytes at most: every batch entry's table has to lie on that grid, not
    the first one's alone."""

    assert _lanes(table_batch=table_batch, table_dtype=table_dtype) == lanes


def test_every_other_stride_is_part_of_the_alignment() -> None:
    assert _lanes() == 1
    for name in ("x_batch", "x_token", "x_head", "grad_batch", "grad_token", "grad_head"):
        assert _lanes(**{name: 8001}) == 8 and _lanes(**{name: 8008}) == 1
    for name in ("x", "grad", "out"):
        assert _lanes(**{name: 4098}) == 8 and _lanes(**{name: 4104}) == 2


def test_a_graph_through_the_norms_backward_is_refused(monkeypatch) -> None:
    """The gradients of heads and norm weights depend on both; without a norm the turn is linear in its gradient."""

    class Library:
        def __getattr__(self, name):
            return lambda *args: 256 if name.endswith("_bytes") else 0

    monkeypatch.setattr(rotary._native, "load", Library)
    monkeypatch.setattr(rotary, "_elsewhere", lambda tensor: False)
    monkeypatch.setattr(rotary, "_stream", lambda tensor: 0)
    q, table, weight = torch.zeros(1, 3, 2, 8).requires_grad_(), torch.zeros(1, 3, 8), torch.ones(8).requires_grad_()
    for wanted, heads, scale in (([q], q, weight.detach()), ([weight], q.detach(), weight), ([q, weight], q, weight)):
        out = rotary.rotary(heads, None, table, q_weight=scale)[0]
        with pytest.raises(RuntimeError, match="graph"):
            torch.autograd.grad(out.sum(), wanted, create_graph=True)
        grads = torch.autograd.grad(rotary.rotary(heads, None, table, q_weight=scale)[0].sum(), wanted)
        assert [g.shape for g in grads] == [t.shape for t in wanted]
    (grad,) = torch.autograd.grad(rotary.rotary(q, None, table)[0].sum(), [q], create_graph=True)
    assert not grad.requires_grad
