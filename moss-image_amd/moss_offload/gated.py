"""The gated activation between the two products of a feed-forward (``csrc/mo_gated.hip``).

``out = act(gate) * cap(up)``: ``"situ"`` is the model's, ``4 tanh(g/4) sigmoid(g) * 25 tanh(u/25)`` (reference
``training/model.py:27-38``, composed there of nine operations that save six tensors of the feed-forward's width);
``"silu"`` is ``g sigmoid(g) * u``. One launch a direction, fp32 inside, each result rounded once. What the backward
pass needs, ``up`` and ``gate``, may be kept in 8 bits, written in the forward's pass.

``up`` and ``gate`` are ``[..., cols]``, dense rows any distance apart, or one tensor ``[..., 2 * cols]`` with ``up``
first, as a fused projection leaves them (``gate=None``).
"""

from __future__ import annotations

import struct

import torch

from . import _native
from ._operands import CODES, elsewhere, first_derivatives, like, pitch, plain, rows, stream
from .kept8 import Kept8, empty

KINDS = ("situ", "silu")
_CALL = struct.Struct("=18Q4I")  # mo_gated_call


def _kind(kind: str) -> bool:
    if kind not in KINDS:
        raise ValueError(f"gated kind must be one of {KINDS}.")
    return kind == "silu"


def _halves(up: torch.Tensor, gate: torch.Tensor | None):
    """(up's matrix, gate's matrix, their addresses, columns, the output's shape)."""

    first = rows(up, "gated up")
    if gate is None:
        if up.shape[-1] % 2:
            raise ValueError("gated takes up and gate side by side in an even last dimension, or both.")
        cols = up.shape[-1] // 2
        return first, first, (first.data_ptr(), first.data_ptr() + cols * first.element_size()), cols, (*up.shape[:-1], cols)
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.get_device() != up.get_device():
        raise ValueError("gated up and gate must have one shape, dtype and device.")
    second = rows(gate, "gated gate")
    return first, second, (first.data_ptr(), second.data_ptr()), up.shape[-1], up.shape


def gated_forward(up: torch.Tensor, gate: torch.Tensor | None = None, *, kind: str = "situ", keep: bool = False):
    """``act(gate) * cap(up)``, contiguous. With ``keep``: ``(out, up, gate)``, the last two as ``Kept8`` of what came
    in (fused: one of ``[..., 2, cols]`` and None), for ``gated_backward``. No graph: ``gated`` has one."""

    lib = _native.load()
    silu = _kind(kind)
    plain("gated", up, gate)
    first, second, addresses, cols, shape = _halves(up, gate)
    if elsewhere(up, "gated"):
        with torch.cuda.device(up.device):
            return gated_forward(up, gate, kind=kind, keep=keep)
    count = first.shape[0]
    out = up.new_empty(shape) if gate is None else like(up)
    kept, kept_gate, places, strides = None, None, (0, 0, 0, 0), (0, 0)
    if keep and gate is None:
        kept = empty((*shape[:-1], 2, cols), up)
        values, groups = kept.values.shape[-1], kept.exponents.shape[-1]
        at, exponents = kept.values.data_ptr(), kept.exponents.data_ptr()
        places, strides = (at, at + values, exponents, exponents + groups), (2 * values, 2 * groups)
    elif keep:
        kept, kept_gate = empty(shape, up), empty(shape, up)
        places = tuple(t.data_ptr() for t in (kept.values, kept_gate.values, kept.exponents, kept_gate.exponents))
        strides = kept.values.shape[-1], kept.exponents.shape[-1]
    if count:
        call = _CALL.pack(
            *addresses, 0, 0, 0, out.data_ptr(), 0, *places, count, pitch(first), pitch(second), 0, cols, *strides, cols,
            CODES[up.dtype], silu, 0)
        _native.check("mo_gated_forward", lib.mo_gated_forward(call, stream(up)))
    return (out, kept, kept_gate) if keep else out


def gated_backward(grad: torch.Tensor, up, gate=None, *, kind: str = "situ"):
    """The gradients of ``gated_forward``'s inputs from its output's: one tensor ``[..., 2 * cols]`` where ``gate`` is
    None (``up`` fused, or the ``Kept8`` of it), else those of ``up`` and ``gate``."""

    lib = _native.load()
    silu = _kind(kind)
    kept, fused = isinstance(up, Kept8), gate is None
    plain("gated", grad, *(t for k in (up, gate) if k is not None for t in ((k.values, k.exponents) if kept else (k,))))
    matrix = rows(grad, "gated gradient")
    count, cols = matrix.shape
    if kept:
        expected = (*grad.shape[:-1], 2, cols) if fused else grad.shape
        for k in (up, gate):
            if k is not None and (not isinstance(k, Kept8) or k.shape != expected or k.dtype != grad.dtype
                                  or k.device != grad.device):
                raise ValueError("gated operands in 8 bits must be of the gradient's shape (fused: [..., 2, cols]), dtype and "
                                 "device.")
        values, groups = up.values.shape[-1], up.exponents.shape[-1]
        if fused:
            at, exponents = up.values.data_ptr(), up.exponents.data_ptr()
            addresses = at, at + values, exponents, exponents + groups
        else:
            addresses = tuple(t.data_ptr() for t in (up.values, gate.values, up.exponents, gate.exponents))
        strides, steps = (0, 0), (values * (1 + fused), groups * (1 + fused))
    else:
        first, second, places, width, shape = _halves(up, gate)
        if shape != grad.shape or up.dtype != grad.dtype or up.get_device() != grad.get_device():
            raise ValueError("gated gradient and operands must have one shape, dtype and device.")
        addresses, strides, steps = (*places, 0, 0), (pitch(first), pitch(second)), (0, 0)
    if elsewhere(grad, "gated"):
        with torch.cuda.device(grad.device):
            return gated_backward(grad, up, gate, kind=kind)
    if fused:
        out = grad.new_empty((*grad.shape[:-1], 2 * cols))
        outs = out.data_ptr(), out.data_ptr() + cols * out.element_size()
    else:
        out = like(grad), like(grad)
        outs = out[0].data_ptr(), out[1].data_ptr()
    if count:
        call = _CALL.pack(
            *addresses, matrix.data_ptr(), *outs, 0, 0, 0, 0, count, *strides, pitch(matrix), cols * (1 + fused), *steps, cols,
            CODES[grad.dtype], silu, 0)
        _native.check("mo_gated_backward", lib.mo_gated_backward(call, stream(grad)))
    return out


class _GatedFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, up, gate, kind, keep, graph):
        if not graph:  # needs_input_grad is set all the same
            return gated_forward(up, gate, kind=kind)
        ctx.kind, ctx.fused, ctx.keep, ctx.dtype = kind, gate is None, keep, up.dtype
        if not keep:
            ctx.save_for_backward(up, gate)
            return gated_forward(up, gate, kind=kind)
        out, *kept = gated_forward(up, gate, kind=kind, keep=True)
        ctx.cols = out.shape[-1]
        ctx.save_for_backward(*(t for k in kept if k is not None for t in (k.values, k.exponents)))
        return out

    @staticmethod
    def backward(ctx, grad):
        first_derivatives("gated")
        saved = ctx.saved_tensors
        if ctx.keep:
            saved = [Kept8(*saved[i : i + 2], ctx.cols, ctx.dtype) for i in range(0, len(saved), 2)]
        grads = gated_backward(grad, *saved, kind=ctx.kind)
        return *((grads, None) if ctx.fused else grads), None, None, None


def gated(up: torch.Tensor, gate: torch.Tensor | None = None, *, kind: str = "situ", keep: bool = False) -> torch.Tensor:
    """``gated_forward`` with its gradients (first derivatives). ``keep``: the backward pass's ``up`` and ``gate`` are
    kept in 8 bits, and the gradients are those at what 8 bits keep of them."""

    return _GatedFunction.apply(up, gate, kind, keep, torch.is_grad_enabled())
