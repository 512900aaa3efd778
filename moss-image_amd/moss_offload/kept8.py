"""Activations in 8 bits between the forward and the backward pass (``csrc/mo_keep.h``, ``csrc/mo_gated.hip``).

A matrix is kept as int8 and a power of two for each 32 values of a row: the smallest, from 2**-126 on, with which
127 reaches the largest of them. Each value is off by at most half a step, 1/127 of its group's largest (2**-127 where
that is less, in groups of the smallest numbers); where a step's 64 is past the type's largest value, by less than a whole one, 1/64.
1 + 1/32 bytes a value, where bfloat16 has two; the offload moves as many fewer bytes. The reference keeps and moves
what autograd saved (``training/activation_offload.py:80-149``).

``keep8`` makes it and ``Kept8.restore`` reads it back; the backward passes of ``norms``, ``gated`` and ``adapters``
read it as it is. ``checkpoint_kept8`` checkpoints a block whose input is kept so.
"""

from __future__ import annotations

import torch

from . import _native
from ._operands import CODES, elsewhere, first_derivatives, like, pitch, plain, rows, stream

GROUP = 32


class Kept8:
    """``values``: int8 ``[..., groups * 32]`` (zeros past ``cols``); ``exponents``: uint8 ``[..., groups]``, biased by
    127 (255: the group held an infinity or a NaN and reads back as NaN); ``dtype``: what it was made from."""

    __slots__ = ("values", "exponents", "cols", "dtype")

    def __init__(self, values: torch.Tensor, exponents: torch.Tensor, cols: int, dtype: torch.dtype) -> None:
        groups = -(-cols // GROUP)
        if values.dtype != torch.int8 or exponents.dtype != torch.uint8 or dtype not in CODES:
            raise TypeError("Kept8 takes int8 values, uint8 exponents and a bfloat16, float16 or float32 dtype.")
        if cols < 1 or values.ndim < 1 or values.shape[-1] != groups * GROUP \
                or exponents.shape != (*values.shape[:-1], groups) or values.get_device() != exponents.get_device():
            raise ValueError("Kept8 values and exponents do not fit its columns, each other or one device.")
        values, exponents = values.contiguous(), exponents.contiguous()
        self.values = values.clone() if values.data_ptr() % 8 else values
        self.exponents, self.cols, self.dtype = exponents, cols, dtype

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.values.shape[:-1], self.cols))

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.exponents.numel()

    def restore(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values it stands for, in ``dtype`` (what it was made from)."""

        lib = _native.load()
        dtype = dtype or self.dtype
        if dtype not in CODES:
            raise TypeError(f"Kept8 restores to bfloat16, float16 or float32 (got {dtype}).")
        plain("Kept8", self.values, self.exponents)
        if elsewhere(self.values, "Kept8"):
            with torch.cuda.device(self.values.device):
                return self.restore(dtype)
        exact = self.cols == self.values.shape[-1]
        out = like(self.values, dtype) if exact else self.values.new_empty(self.shape, dtype=dtype)
        if out.numel():
            _native.check("mo_keep_restore", lib.mo_keep_restore(
                self.values.data_ptr(), self.exponents.data_ptr(), out.data_ptr(), CODES[dtype],
                out.numel() // self.cols, self.cols, self.cols, stream(out)))
        return out


def empty(shape, tensor: torch.Tensor) -> Kept8:
    """Room for a kernel to write a tensor of ``shape``, and ``tensor``'s type, in 8 bits."""

    kept = Kept8.__new__(Kept8)
    groups = -(-shape[-1] // GROUP)
    if shape == tensor.shape and shape[-1] % GROUP == 0:
        kept.values = like(tensor, torch.int8)
    else:
        kept.values = tensor.new_empty((*shape[:-1], groups * GROUP), dtype=torch.int8)
    kept.exponents = tensor.new_empty((*shape[:-1], groups), dtype=torch.uint8)
    kept.cols, kept.dtype = shape[-1], tensor.dtype
    return kept


def keep8(x: torch.Tensor) -> Kept8:
    """``x``, bfloat16, float16 or float32 ``[..., cols]``, in 8 bits. It carries no graph."""

    lib = _native.load()
    plain("keep8", x)
    matrix = rows(x, "keep8's tensor")
    if elsewhere(x, "keep8"):
        with torch.cuda.device(x.device):
            return keep8(x)
    kept = empty(x.shape, x)
    if matrix.shape[0]:
        _native.check("mo_keep_pack", lib.mo_keep_pack(
            matrix.data_ptr(), CODES[x.dtype], matrix.shape[0], matrix.shape[1], pitch(matrix), kept.values.data_ptr(),
            kept.exponents.data_ptr(), stream(x)))
    return kept


# ---- a checkpointed block whose input is kept in 8 bits -------------------------------------------------


def _not_captured(tensor: torch.Tensor) -> None:
    if tensor.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("checkpoint_kept8 cannot be captured into a graph.")


class _CheckpointFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, function, tokens, *others):
        kept, kind = keep8(tokens), tokens.device.type
        ctx.function, ctx.dtype, ctx.cols, ctx.kind = function, tokens.dtype, tokens.shape[-1], kind
        ctx.autocast = {"enabled": torch.is_autocast_enabled(kind), "dtype": torch.get_autocast_dtype(kind), "cache_enabled": False}
        ctx.random = torch.get_rng_state(), torch.cuda.get_rng_state(tokens.device)
        ctx.others = [None if isinstance(t, torch.Tensor) else t for t in others]
        ctx.places = [i for i, t in enumerate(others) if isinstance(t, torch.Tensor)]
        ctx.wanted = [t.requires_grad for t in others if isinstance(t, torch.Tensor)]
        ctx.save_for_backward(kept.values, kept.exponents, *(others[i] for i in ctx.places))
        # without autocast's cache, in both runs: what is cast here has no graph, and whoever found it there, the second run
        # or a layer's next use in the same region, would lose the weights' gradients
        with torch.autocast(kind, **ctx.autocast):
            out = function(tokens, *others)
        if not isinstance(out, torch.Tensor):
            raise TypeError("checkpoint_kept8 takes a function that returns one tensor.")
        return out

    @staticmethod
    def backward(ctx, gradient):
        first_derivatives("checkpoint_kept8")
        _not_captured(gradient)
        values, exponents, *given = ctx.saved_tensors
        tokens = Kept8(values, exponents, ctx.cols, ctx.dtype).restore().requires_grad_(ctx.needs_input_grad[1])
        others = list(ctx.others)
        leaves = [tokens]
        for place, tensor, wanted in zip(ctx.places, given, ctx.wanted):
            others[place] = tensor.detach().requires_grad_(wanted)
            leaves.append(others[place])
        with torch.random.fork_rng([tokens.device]):
            torch.set_rng_state(ctx.random[0])
            torch.cuda.set_rng_state(ctx.random[1], tokens.device)
            with torch.enable_grad(), torch.autocast(ctx.kind, **ctx.autocast):
                out = ctx.function(tokens, *others)
        if out.requires_grad:
            torch.autograd.backward(out, gradient)
        grads = [None] * len(others)
        for place, leaf in zip(ctx.places, leaves[1:]):
            grads[place] = leaf.grad
        return None, tokens.grad, *grads


def checkpoint_kept8(function, tokens: torch.Tensor, *others) -> torch.Tensor:
    """``function(tokens, *others)``, one tensor, of which the backward pass keeps ``tokens`` in 8 bits and computes
    the rest again from that: the result is the exact input's, the gradients are taken at what 8 bits keep of it.

    As with a reentrant checkpoint, the parameters inside get their gradients by accumulation (``backward()``, not
    ``torch.autograd.grad``), and an input must want a gradient: the function's parameters alone are not seen. Neither
    pass while a graph is captured: the random numbers' state, which the second run starts from, cannot be had then."""

    if not torch.is_grad_enabled():
        return function(tokens, *others)
    if not any(isinstance(t, torch.Tensor) and t.requires_grad for t in (tokens, *others)):
        raise RuntimeError("checkpoint_kept8 needs an input that requires grad.")
    _not_captured(tokens)
    return _CheckpointFunction.apply(function, tokens, *others)
