"""Low-rank adapters of many requests at once beside a shared projection (``csrc/mo_adapters.hip``).

``y = result + scale_i * (x @ a_i.T) @ b_i.T``, ``result`` the shared projection's and ``i`` the adapter of the request
that a row belongs to. With one request and one adapter it is the reference's LoRA linear (``training/lora.py:60-86``);
a packed batch may bring an adapter for each sample, a batch of sampling requests one for each row. The products in
between stay in fp32 and ``y`` is rounded once. The gradients read ``x`` or what 8 bits keep of it.

Rows are ``[..., features]``, dense, any distance apart; ranks go up to 128. The requests are the first dimension of an ``x`` of
three or more (one of two is one request), or ``cu_seqlens`` (``[requests + 1]``) says which rows each has; ``index`` (``[requests]``) says which adapter, any number
outside ``[0, adapters)`` none. Rows without an adapter pass ``result`` on. Without an index request ``i`` has
adapter ``i``, or the only one.
"""

from __future__ import annotations

import struct

import torch

from . import _native
from ._operands import CODES, elsewhere, first_derivatives, like as _like, pitch, plain, stream, whole
from ._operands import rows as _dense_rows
from .kept8 import Kept8, keep8

MAX_RANK = 128
MAX_STRIDE = 1 << 22
_CALL = struct.Struct("=20Q6IfI")  # mo_adapters_call


def rows(tensor: torch.Tensor, what: str) -> torch.Tensor:
    """``_operands.rows``, near enough to each other for the kernels' 32-bit offsets."""

    matrix = _dense_rows(tensor, what)
    return matrix.contiguous() if matrix.shape[0] > 1 and matrix.stride(0) > MAX_STRIDE else matrix


def _address(tensor: torch.Tensor | None) -> int:
    return 0 if tensor is None else tensor.data_ptr()


def _check(like, shape, a, b, scale, cu_seqlens, index):
    """(a, b, scale tensor, factor, cu_seqlens, index, requests) of a call on rows whose shape begins with ``shape``."""

    if a.ndim != 3 or b.ndim != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or not a.numel() or not b.numel():
        raise ValueError("adapters must be a [adapters, rank, in] and b [adapters, out, rank], not empty.")
    if a.shape[1] > MAX_RANK:
        raise ValueError(f"adapters have ranks up to {MAX_RANK} (got {a.shape[1]}).")
    if a.dtype != like.dtype or b.dtype != like.dtype or a.get_device() != like.get_device() \
            or b.get_device() != like.get_device():
        raise ValueError("adapters must be of the tokens' dtype, on their device.")
    count, factor = a.shape[0], 1.0
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != (count,) or scale.get_device() != like.get_device():
            raise ValueError("adapters' scale must be a number, or float32 [adapters] on the tokens' device.")
        scale = scale.contiguous()
    else:
        scale, factor = None, float(scale)
    requests = 1 if len(shape) < 2 else shape[0]
    if cu_seqlens is not None:
        if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 2:
            raise ValueError("adapters' cu_seqlens must be [requests + 1].")
        requests = cu_seqlens.shape[0] - 1
        cu_seqlens = whole(cu_seqlens, requests + 1, like, "adapters' cu_seqlens")
    elif index is None and count == 1:
        requests = 1
    index = whole(index, requests, like, "adapters' index")
    if index is None and count not in (1, requests):
        raise ValueError("adapters need an index where the requests are not as many.")
    return a.contiguous(), b.contiguous(), scale, factor, cu_seqlens, index, requests


def _space(lib, call, backward: bool, like: torch.Tensor):
    # freed to the caching allocator after the call; stream order keeps it alive for the kernels
    nbytes = lib.mo_adapters_workspace_bytes(call, backward)
    return (like.new_empty(nbytes, dtype=torch.uint8), nbytes) if nbytes else (None, 0)


def adapters_forward(x: torch.Tensor, result: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale=1.0, *,
                     cu_seqlens: torch.Tensor | None = None, index: torch.Tensor | None = None, hidden: bool = False):
    """``result + scale_i * (x @ a_i.T) @ b_i.T``, contiguous. ``x``: ``[..., in]``; ``result``: ``[..., out]``; ``a``:
    ``[adapters, rank, in]``; ``b``: ``[adapters, out, rank]``, all of one type; ``scale``: a number, or float32
    ``[adapters]``. With ``hidden``: ``(y, x @ a_i.T)``, the latter float32 ``[rows, rank]``, for ``adapters_backward``.
    No graph: ``adapters`` has one."""

    lib = _native.load()
    plain("adapters", x, result, a, b, cu_seqlens, index, scale if isinstance(scale, torch.Tensor) else None)
    tokens, base = rows(x, "adapters' tokens"), rows(result, "adapters' result")
    a, b, scales, factor, cu, which, requests = _check(x, x.shape[:-1] if x.ndim > 2 else (1,), a, b, scale, cu_seqlens, index)
    count, features = tokens.shape
    if x.shape[:-1] != result.shape[:-1] or result.dtype != x.dtype or result.get_device() != x.get_device() \
            or a.shape[2] != features or b.shape[1] != base.shape[1]:
        raise ValueError("adapters' tokens and result must have the same rows, dtype and device, and the adapters' features.")
    if elsewhere(x, "adapters"):
        with torch.cuda.device(x.device):
            return adapters_forward(x, result, a, b, scale, cu_seqlens=cu_seqlens, index=index, hidden=hidden)
    rank = a.shape[1]
    y = _like(result)
    between = x.new_empty((count, rank), dtype=torch.float32)
    if count:
        call = _CALL.pack(
            tokens.data_ptr(), 0, base.data_ptr(), y.data_ptr(), a.data_ptr(), b.data_ptr(), _address(scales), _address(cu),
            _address(which), between.data_ptr(), 0, 0, 0, 0, 0, count, pitch(tokens), pitch(base), 0, 0, requests, a.shape[0],
            rank, features, base.shape[1], CODES[x.dtype], factor, 0)
        space, nbytes = _space(lib, call, False, x)
        _native.check("mo_adapters_forward",
                      lib.mo_adapters_forward(call, _address(space), nbytes, stream(x)))
    return (y, between) if hidden else y


def _backward(grad, x, hidden, a, b, scale, cu_seqlens, index, add, wanted):
    lib = _native.load()
    kept = isinstance(x, Kept8)
    plain("adapters", grad, hidden, a, b, cu_seqlens, index, add, scale if isinstance(scale, torch.Tensor) else None,
          *((x.values, x.exponents) if kept else (x,)))
    matrix = rows(grad, "adapters' gradient")
    lead = grad.shape[:-1] if grad.ndim > 2 else (1,)
    a, b, scales, factor, cu, which, requests = _check(grad, lead, a, b, scale, cu_seqlens, index)
    count, out_features = matrix.shape
    rank, in_features = a.shape[1:]
    if b.shape[1] != out_features or hidden.dtype != torch.float32 or hidden.shape != (count, rank) \
            or hidden.get_device() != grad.get_device():
        raise ValueError("adapters' gradient must have b's features, and hidden be the forward pass's: float32 [rows, rank].")
    for tensor in (x, add):
        if tensor is not None and (tensor.shape != (*grad.shape[:-1], in_features) or tensor.dtype != grad.dtype
                                   or tensor.device != grad.device):
            raise ValueError("adapters' tokens must have the gradient's rows, dtype and device, and a's features.")
    if elsewhere(grad, "adapters"):
        with torch.cuda.device(grad.device):
            return _backward(grad, x, hidden, a, b, scale, cu_seqlens, index, add, wanted)
    source = None if x is None else x.values if kept else rows(x, "adapters' tokens")
    hidden = hidden.contiguous()
    added = None if add is None else rows(add, "adapters' add")
    dx = grad.new_empty((*grad.shape[:-1], in_features)) if wanted[0] else None
    da, db = (_like(t) if w else None for t, w in zip((a, b), wanted[1:]))
    if count and any(wanted):
        call = _CALL.pack(
            _address(source), x.exponents.data_ptr() if kept else 0, 0, 0, a.data_ptr(), b.data_ptr(), _address(scales),
            _address(cu), _address(which), hidden.data_ptr(), matrix.data_ptr(), _address(added), _address(dx), _address(da),
            _address(db), count, 0 if kept or source is None else pitch(source), 0, pitch(matrix),
            0 if added is None else pitch(added), requests, a.shape[0], rank, in_features, out_features, CODES[grad.dtype],
            factor, 0)
        space, nbytes = _space(lib, call, True, grad)
        _native.check("mo_adapters_backward",
                      lib.mo_adapters_backward(call, _address(space), nbytes, stream(grad)))
    else:
        for t in (da, db):
            if t is not None:
                t.zero_()
    return dx, da, db


def adapters_backward(grad: torch.Tensor, x, hidden: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale=1.0, *,
                      cu_seqlens: torch.Tensor | None = None, index: torch.Tensor | None = None,
                      add: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(d x, d a, d b)`` from ``y``'s gradient (``result``'s is that gradient itself): ``x`` the forward pass's, or a
    ``Kept8`` of it, ``hidden`` what that pass gave. ``add``: the shared projection's input gradient, added to ``d x``
    before its rounding. Sums over the rows are fp32, in a fixed order; an adapter that no row has gets zeros."""

    return _backward(grad, x, hidden, a, b, scale, cu_seqlens, index, add, (True, True, True))


class _AdaptersFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, result, a, b, scale, cu_seqlens, index, keep, graph):
        how = {"cu_seqlens": cu_seqlens, "index": index}
        if not graph:  # needs_input_grad is set all the same
            return adapters_forward(x, result, a, b, scale, **how)
        y, hidden = adapters_forward(x, result, a, b, scale, hidden=True, **how)
        ctx.tensor_scale = isinstance(scale, torch.Tensor)
        ctx.number = None if ctx.tensor_scale else scale
        ctx.cols, ctx.dtype, ctx.kept = x.shape[-1], x.dtype, False
        saved = (None, None)
        if ctx.needs_input_grad[2]:
            ctx.kept = bool(keep) or isinstance(keep, Kept8)
            kept = keep if isinstance(keep, Kept8) else keep8(x) if keep else None
            saved = (kept.values, kept.exponents) if ctx.kept else (x, None)
        ctx.save_for_backward(*saved, hidden if ctx.needs_input_grad[3] else None, a, b,
                              scale if ctx.tensor_scale else None, cu_seqlens, index)
        ctx.rows = hidden.shape
        return y

    @staticmethod
    def backward(ctx, grad):
        first_derivatives("adapters")
        x, exponents, hidden, a, b, scale, cu_seqlens, index = ctx.saved_tensors
        if ctx.kept:
            x = Kept8(x, exponents, ctx.cols, ctx.dtype)
        needed = ctx.needs_input_grad
        wanted = needed[0], needed[2], needed[3]
        if hidden is None:  # d b's alone
            hidden = torch.empty(ctx.rows, dtype=torch.float32, device=grad.device)
        dx, da, db = _backward(grad, x, hidden, a, b, scale if ctx.tensor_scale else ctx.number, cu_seqlens, index, None, wanted) \
            if any(wanted) else (None, None, None)
        return dx, grad if needed[1] else None, da, db, None, None, None, None, None


def adapters(x: torch.Tensor, result: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale=1.0, *,
             cu_seqlens: torch.Tensor | None = None, index: torch.Tensor | None = None, keep=False) -> torch.Tensor:
    """``adapters_forward`` with gradients for the tokens, the result and the adapters (first derivatives; none for the
    scales). ``a``, ``b``: also ``[rank, in]`` and ``[out, rank]``, one adapter. ``keep``: True, or a ``Kept8`` of ``x`` that
    several projections share: ``d a`` is taken from what 8 bits keep of ``x``."""

    if isinstance(scale, torch.Tensor) and scale.requires_grad:
        raise RuntimeError("adapters have no gradient for their scales.")
    if isinstance(keep, Kept8) and (keep.shape != x.shape or keep.dtype != x.dtype or keep.device != x.device):
        raise ValueError("adapters' kept tokens must have the tokens' shape, dtype and device.")
    if a.ndim == 2 and b.ndim == 2:
        a, b = a.unsqueeze(0), b.unsqueeze(0)
    return _AdaptersFunction.apply(x, result, a, b, scale, cu_seqlens, index, keep, torch.is_grad_enabled())
