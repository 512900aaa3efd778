"""Layer and RMS norms of rows, with a weight, a bias and a modulation for each sample (``csrc/mo_norm.hip``).

``out = ((x - mean) / sqrt(variance + eps) * weight + bias) * (1 + scale) + shift``; an RMS norm takes the mean as
zero. The reference norms and modulates with composed operations (``training/model.py:154-172``, ``:291-314``), which
read and write the tokens once for each and save several copies of them. Here the forward pass is one launch and the
backward pass two or three, fp32 inside, each result rounded once, and the input may be kept in 8 bits in between.

Rows are ``[..., dim]``, dense, any distance apart, up to 16384 values. ``scale`` and ``shift`` are ``[samples, dim]``:
``x``'s first dimension is the samples, or ``cu_seqlens`` (``[samples + 1]``) says which rows each has; rows in no
sample give zeros, get a gradient of zero and take part in no sum.
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import _native
from ._operands import CODES, elsewhere, first_derivatives, like as _like, pitch, plain, rows, stream, whole
from .kept8 import Kept8, empty

KINDS = ("layer", "rms")
MAX_DIM = 16384
_CALL = struct.Struct("=21Q6IfI")  # mo_norm_call


class NormGradients(NamedTuple):
    x: torch.Tensor
    weight: torch.Tensor | None
    bias: torch.Tensor | None
    scale: torch.Tensor | None
    shift: torch.Tensor | None


def _address(tensor: torch.Tensor | None) -> int:
    return 0 if tensor is None else tensor.data_ptr()


def _pair(first, second, shape, like, names):
    """Two vectors or stacks of them of one type, last dimension dense, and that type's code."""

    code, out = None, []
    for tensor, name in zip((first, second), names):
        if tensor is not None:
            if tensor.dtype not in CODES or tensor.shape != shape or tensor.get_device() != like.get_device() \
                    or code not in (None, tensor.dtype):
                raise ValueError(f"norm {names[0]} and {names[1]} must be {list(shape)}, of one floating type, on the "
                                 "rows' device.")
            code = tensor.dtype
            if tensor.stride(-1) != 1 and shape[-1] > 1:
                tensor = tensor.contiguous()
        out.append(tensor)
    return out[0], out[1], 2 if code is None else CODES[code]


def _check(like, shape, kind, weight, bias, scale, shift, cu_seqlens):
    """(samples, weight, bias, their type, scale, shift, their type, cu_seqlens) of a call on rows of ``shape``."""

    if kind not in KINDS:
        raise ValueError(f"norm kind must be one of {KINDS}.")
    if not shape or not 1 <= shape[-1] <= MAX_DIM:
        raise ValueError(f"norm rows must be [..., dim] of 1 to {MAX_DIM} values.")
    dim = shape[-1]
    weight, bias, weight_code = _pair(weight, bias, (dim,), like, ("weight", "bias"))
    given = scale if scale is not None else shift
    if given is None:
        if cu_seqlens is not None:
            raise ValueError("norm cu_seqlens go with a scale or a shift.")
        return 0, weight, bias, weight_code, None, None, 2, None
    if given.ndim != 2 or not given.shape[0] and shape[:-1].numel():
        raise ValueError("norm scale and shift must be [samples, dim].")
    samples = given.shape[0]
    scale, shift, scale_code = _pair(scale, shift, (samples, dim), like, ("scale", "shift"))
    if cu_seqlens is not None:
        cu_seqlens = whole(cu_seqlens, samples + 1, like, "norm cu_seqlens")
    elif samples != 1 and (len(shape) < 2 or shape[0] != samples):
        raise ValueError("norm scale and shift must have one row for each of x's first dimension, or cu_seqlens.")
    return samples, weight, bias, weight_code, scale, shift, scale_code, cu_seqlens


def _run(name, lib, call, like):
    if name == "mo_norm_forward":
        return _native.check(name, lib.mo_norm_forward(call, stream(like)))
    nbytes = lib.mo_norm_workspace_bytes(call)
    # freed to the caching allocator after the call; stream order keeps it alive for the kernels
    space = like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _native.check(name, lib.mo_norm_backward(call, _address(space), nbytes, stream(like)))


def norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                 kind: str = "rms", scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
                 cu_seqlens: torch.Tensor | None = None, eps: float = 1e-6, stats: bool = False, keep: bool = False):
    """The normed rows, contiguous, in ``x``'s type. ``weight``, ``bias``: ``[dim]``; ``scale``, ``shift``:
    ``[samples, dim]``. With ``stats`` or ``keep``: ``(out, stats, kept)``: for each row its mean and 1 / deviation, fp32
    ``[rows, 2]``, and ``x`` in 8 bits, made in the same pass; None for the one not asked for. No graph: ``norm`` has one."""

    lib = _native.load()
    plain("norm", x, weight, bias, scale, shift, cu_seqlens)
    matrix = rows(x, "norm rows")
    samples, weight, bias, weight_code, scale, shift, scale_code, cu = \
        _check(x, x.shape, kind, weight, bias, scale, shift, cu_seqlens)
    if elsewhere(x, "norm"):
        with torch.cuda.device(x.device):
            return norm_forward(x, weight, bias, kind=kind, scale=scale, shift=shift, cu_seqlens=cu, eps=eps, stats=stats,
                                keep=keep)
    count, dim = matrix.shape
    out = _like(x)
    statistics = x.new_empty((count, 2), dtype=torch.float32) if stats else None
    kept = empty(x.shape, x) if keep else None
    if count:
        _run("mo_norm_forward", lib, _CALL.pack(
            matrix.data_ptr(), 0, 0, out.data_ptr(), _address(statistics), _address(weight), _address(bias), _address(scale),
            _address(shift), kept.values.data_ptr() if keep else 0, kept.exponents.data_ptr() if keep else 0, 0, 0, 0, 0,
            _address(cu), count, pitch(matrix), 0, 0 if scale is None else scale.stride(0),
            0 if shift is None else shift.stride(0), samples, dim, CODES[x.dtype], weight_code, scale_code,
            kind == "layer", eps, 0), x)
    return (out, statistics, kept) if stats or keep else out


def _backward(grad, x, stats, weight, bias, kind, scale, shift, cu_seqlens, wanted) -> NormGradients:
    lib = _native.load()
    kept = isinstance(x, Kept8)
    plain("norm", grad, stats, weight, bias, scale, shift, cu_seqlens, *((x.values, x.exponents) if kept else (x,)))
    matrix = rows(grad, "norm gradient")
    count, dim = matrix.shape
    if grad.shape != x.shape or grad.dtype != x.dtype or grad.get_device() != x.device.index:
        raise ValueError("norm gradient and rows must have one shape, dtype and device.")
    if stats.dtype != torch.float32 or stats.shape != (count, 2) or stats.get_device() != grad.get_device():
        raise ValueError("norm stats must be the forward pass's: float32 [rows, 2].")
    samples, weight, bias, weight_code, scale, shift, scale_code, cu = \
        _check(grad, grad.shape, kind, weight, bias, scale, shift, cu_seqlens)
    if elsewhere(grad, "norm"):
        with torch.cuda.device(grad.device):
            return _backward(grad, x, stats, weight, bias, kind, scale, shift, cu, wanted)
    source = x.values if kept else rows(x, "norm rows")
    stats = stats.contiguous()
    stats = stats.clone() if stats.data_ptr() % 8 else stats
    out = _like(grad)
    # the sums are as wide as their tensors; with no rows they are zero
    grads = [_like(t) if t is not None and w else None
             for t, w in zip((weight, bias, scale, shift), wanted)]
    if count:
        _run("mo_norm_backward", lib, _CALL.pack(
            source.data_ptr(), x.exponents.data_ptr() if kept else 0, matrix.data_ptr(), out.data_ptr(), stats.data_ptr(),
            _address(weight), _address(bias), _address(scale), _address(shift), 0, 0, *map(_address, grads), _address(cu), count,
            0 if kept else pitch(source), pitch(matrix), 0 if scale is None else scale.stride(0),
            0 if shift is None else shift.stride(0), samples, dim, CODES[grad.dtype], weight_code, scale_code, kind == "layer",
            0.0, 0), grad)
    else:
        for g in grads:
            if g is not None:
                g.zero_()
    return NormGradients(out, *grads)


def norm_backward(grad: torch.Tensor, x, stats: torch.Tensor, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *, kind: str = "rms", scale: torch.Tensor | None = None,
                  shift: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None) -> NormGradients:
    """The gradients of ``norm_forward``'s arguments from its output's: ``x`` is the forward pass's, or a ``Kept8`` of
    it, ``stats`` what that pass gave. Sums over the rows are fp32, added in a fixed order, in their tensors' types."""

    return _backward(grad, x, stats, weight, bias, kind, scale, shift, cu_seqlens, (True, True, True, True))


class _NormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, shift, cu_seqlens, kind, eps, keep, graph):
        how = {"kind": kind, "scale": scale, "shift": shift, "cu_seqlens": cu_seqlens, "eps": eps}
        if not graph:  # needs_input_grad is set all the same
            return norm_forward(x, weight, bias, **how)
        out, stats, kept = norm_forward(x, weight, bias, stats=True, keep=keep, **how)
        ctx.kind, ctx.cols, ctx.dtype, ctx.keep = kind, x.shape[-1], x.dtype, keep
        saved = (kept.values, kept.exponents) if keep else (x, None)
        ctx.save_for_backward(*saved, stats, weight, bias, scale, shift, cu_seqlens)
        return out

    @staticmethod
    def backward(ctx, grad):
        first_derivatives("norm")
        x, exponents, stats, weight, bias, scale, shift, cu_seqlens = ctx.saved_tensors
        if ctx.keep:
            x = Kept8(x, exponents, ctx.cols, ctx.dtype)
        grads = _backward(grad, x, stats, weight, bias, ctx.kind, scale, shift, cu_seqlens, ctx.needs_input_grad[1:5])
        return *grads, None, None, None, None, None


def norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, kind: str = "rms",
         scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
         eps: float = 1e-6, keep: bool = False) -> torch.Tensor:
    """``norm_forward`` with gradients for all of its tensors (first derivatives). ``keep``: what the backward pass needs of
    ``x`` is kept in 8 bits, and the gradients are those at what 8 bits keep of it."""

    return _NormFunction.apply(x, weight, bias, scale, shift, cu_seqlens, kind, eps, keep, torch.is_grad_enabled())
