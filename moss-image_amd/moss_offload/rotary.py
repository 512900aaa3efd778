"""Rotary positions of attention heads on hand-written kernels (``csrc/mo_rotary.hip``), with the heads'
RMS norm in the same pass where a block has one.

The reference turns queries and keys with composed operations (``training/model.py:41-56`` after the
norms ``:154-172``; the angles ``:136-151``), a dozen launches a side that each round to the tokens' type.
Here a table of sines and cosines is made in one launch (``rotary_table``), and both sides' norms and turns
take one launch, forward (``rotary_forward``) or backward (``rotary_backward``); ``rotary`` has both under
autograd. Everything is fp32 inside and rounded once.

Heads are ``[batch, tokens, heads, head_dim]`` with any strides but a dense last dimension (views of a
fused projection are fine); queries and keys may have different numbers of heads. A table is ``[batch or
1, tokens, rotary_dim]``: half sines, half cosines. ``layout="half"`` pairs value ``i`` with ``i +
rotary_dim / 2`` (the reference's), ``"interleaved"`` neighbours. Values past ``rotary_dim`` are passed on.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _native
from .quant_kernels import _by_address

LAYOUTS = ("half", "interleaved")
SCALINGS = ("linear", "ntk", "yarn")
MAX_HEAD_DIM = 512
_CODES = _native.DTYPE_CODES


def _elsewhere(tensor: torch.Tensor) -> bool:
    """Whether the tensor's device is not the current one, which kernels are launched on."""

    index = tensor.get_device()
    if index < 0:
        raise RuntimeError("rotary operands must be on a HIP device.")
    return index != torch._C._cuda_getDevice()


def _stream(tensor: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(tensor.get_device())


def _plain(*operands: torch.Tensor | None) -> None:
    if not _by_address(*operands):
        raise RuntimeError("rotary operands must be plain tensors without a graph or a tangent; rotary has a gradient.")


def scaled_bands(bands: torch.Tensor, factor: float, method: str = "yarn", *, original_length: int = 4096,
                 slow: float = 1.0, fast: float = 32.0) -> tuple[torch.Tensor, float]:
    """``(bands, amplitude)`` for contexts ``factor`` times the trained length.

    - ``linear``: every band divided by the factor (positions are interpolated);
    - ``ntk``: a larger base: the first band stays, the last is divided by the factor;
    - ``yarn``: bands that turn ``fast`` times or more over ``original_length`` stay, those that turn at
      most ``slow`` times are divided, those between are blended, and the table gets the amplitude
      ``0.1 ln(factor) + 1``.
    """

    if method not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}.")
    if bands.ndim != 1 or not bands.numel() or not math.isfinite(factor) or factor < 1.0:
        raise ValueError("bands must be a vector and the factor at least 1.")
    wide = bands.double()
    amplitude = 1.0
    if method == "linear":
        wide = wide / factor
    elif method == "ntk":
        index = torch.arange(bands.numel(), device=bands.device, dtype=torch.float64)
        wide = wide * factor ** (-index / max(bands.numel() - 1, 1))
    else:
        if not 0.0 <= slow < fast or original_length < 1:
            raise ValueError("yarn needs 0 <= slow < fast and a length of at least 1.")
        keep = ((original_length * wide / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        wide = wide / factor * (1 - keep) + wide * keep
        amplitude = 0.1 * math.log(factor) + 1.0
    return wide.to(bands.dtype), amplitude


def rotary_table(coordinates: torch.Tensor, bands: torch.Tensor, *, amplitude: float = 1.0,
                 dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``[..., tokens, 2 * axes * bands]``: the sines of ``coordinate * band`` (float32 products), axis by axis,
    then the cosines, each times ``amplitude``. ``coordinates``: float32 ``[..., tokens, axes]``; ``bands``:
    float32 ``[bands]``. One axis is a text position; the model's images have four."""

    lib = _native.load()
    _plain(coordinates, bands)
    if coordinates.dtype != torch.float32 or bands.dtype != torch.float32 or dtype not in _CODES:
        raise TypeError("rotary coordinates and bands must be float32, the table bfloat16, float16 or float32.")
    if coordinates.ndim < 2 or bands.ndim != 1 or not coordinates.shape[-1] or not bands.numel():
        raise ValueError("rotary coordinates must be [..., tokens, axes] and bands a vector, neither empty.")
    if bands.get_device() != coordinates.get_device():
        raise RuntimeError("rotary coordinates and bands must be on one device.")
    coordinates, bands = coordinates.contiguous(), bands.contiguous()
    if _elsewhere(coordinates):
        with torch.cuda.device(coordinates.device):
            return rotary_table(coordinates, bands, amplitude=amplitude, dtype=dtype)
    axes = coordinates.shape[-1]
    rows = coordinates.numel() // axes
    out = torch.empty((*coordinates.shape[:-1], 2 * axes * bands.numel()), dtype=dtype, device=coordinates.device)
    if rows:
        _native.check("mo_rotary_table", lib.mo_rotary_table(
            coordinates.data_ptr(), bands.data_ptr(), out.data_ptr(), _CODES[dtype], rows, axes, bands.numel(),
            amplitude, _stream(coordinates)))
    return out


def _heads(tensor: torch.Tensor, like: torch.Tensor, what: str) -> torch.Tensor:
    if tensor.ndim != 4 or tensor.dtype != like.dtype or tensor.get_device() != like.get_device() \
            or tensor.shape[:2] != like.shape[:2] or tensor.shape[3] != like.shape[3]:
        raise ValueError(f"rotary {what} must be [batch, tokens, heads, head_dim] of the queries' batch, tokens, "
                         "head_dim, dtype and device.")
    return tensor if tensor.stride(3) == 1 else tensor.contiguous()


_SIDE, _REST = struct.Struct("=5Q6qII"), struct.Struct("=QQ8IfI")  # mo_rotary_side; mo_rotary_call after its sides
_NO_SIDE = bytes(_SIDE.size)


def _call(sides, table, layout, weights, eps, backward):
    """The call's description, and what it keeps alive, its outputs and weight gradients. ``sides``: (heads or
    None, gradient or None) of queries and keys."""

    if layout not in LAYOUTS:
        raise ValueError(f"rotary layout must be one of {LAYOUTS}.")
    (q, grad_q), (k, grad_k) = sides
    like = next((t for t in (grad_q, grad_k, q, k) if t is not None), None)
    if like is None:
        raise ValueError("rotary needs queries or keys.")
    _plain(table, *weights, q, grad_q, k, grad_k)
    code, table_code = _CODES.get(like.dtype), _CODES.get(table.dtype)
    if code is None or table_code is None:
        raise TypeError("rotary heads and table must be bfloat16, float16 or float32.")
    if like.ndim != 4:
        raise ValueError("rotary heads must be [batch, tokens, heads, head_dim].")
    batch, tokens, _, head_dim = like.shape
    if table.ndim == 2:
        table = table.unsqueeze(0)
    if table.ndim != 3 or table.shape[0] not in (1, batch) or table.shape[1] != tokens:
        raise ValueError("rotary table must be [batch or 1, tokens, rotary_dim].")
    rotary_dim = table.shape[2]
    if head_dim % 2 or not 2 <= head_dim <= MAX_HEAD_DIM or rotary_dim % 2 or not 2 <= rotary_dim <= head_dim:
        raise ValueError(f"rotary needs an even head_dim up to {MAX_HEAD_DIM} and an even rotary_dim up to head_dim.")
    if table.get_device() != like.get_device():
        raise RuntimeError("rotary heads and table must be on one device.")
    table = table.contiguous()
    kept, outs, weight_grads, packed, weight_dtype = [table], [], [], [], None
    for (x, grad), weight in zip(sides, weights):
        given = grad if backward else x
        if given is None:
            outs.append(None)
            weight_grads.append(None)
            packed.append(_NO_SIDE)
            continue
        given = _heads(given, like, "heads")
        out = torch.empty(given.shape, dtype=given.dtype, device=given.device)
        heads = given.shape[2]
        weight_grad = None
        if weight is not None:
            if weight.shape != (head_dim,) or weight.dtype not in _CODES or weight.get_device() != like.get_device() \
                    or weight_dtype not in (None, weight.dtype):
                raise ValueError("rotary norm weights must be [head_dim], of one floating type, on the heads' device.")
            weight_dtype, weight = weight.dtype, weight.contiguous()
            if backward:
                if x is None:
                    raise ValueError("the norm's gradient needs the queries or keys that went in.")
                x = _heads(x, like, "heads")
                if x.shape != given.shape:
                    raise ValueError("rotary gradient and heads must have one shape.")
                weight_grad = torch.empty_like(weight) if heads else torch.zeros_like(weight)
        source = x if backward and weight is not None else None if backward else given
        kept += [given, source, weight]
        packed.append(_SIDE.pack(
            0 if source is None else source.data_ptr(), given.data_ptr() if backward else 0, out.data_ptr(),
            0 if weight is None else weight.data_ptr(), 0 if weight_grad is None else weight_grad.data_ptr(),
            *((0, 0, 0) if source is None else source.stride()[:3]), *(given.stride()[:3] if backward else (0, 0, 0)),
            heads, 0))
        outs.append(out)
        weight_grads.append(weight_grad)
    rest = _REST.pack(table.data_ptr(), 0 if table.shape[0] == 1 else tokens * rotary_dim, code, table_code,
                      _CODES[weight_dtype or torch.float32], batch, tokens, head_dim, rotary_dim,
                      layout == "interleaved", eps, 0)
    call = _native.MoRotaryCall.from_buffer_copy(packed[0] + packed[1] + rest)
    return call, kept, outs, weight_grads, like


def _any(outs) -> bool:
    return any(out is not None and out.numel() for out in outs)


def rotary_forward(q: torch.Tensor | None, k: torch.Tensor | None, table: torch.Tensor, *, layout: str = "half",
                   q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                   eps: float = 1e-6) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The turned queries and keys, contiguous; either side may be None. ``q_weight``, ``k_weight``: ``[head_dim]``
    scales of an RMS norm over each head before the turn (None: no norm). No graph: ``rotary`` has one."""

    lib = _native.load()
    call, _kept, outs, _, like = _call(((q, None), (k, None)), table, layout, (q_weight, k_weight), eps, False)
    if _elsewhere(like):
        with torch.cuda.device(like.device):
            return rotary_forward(q, k, table, layout=layout, q_weight=q_weight, k_weight=k_weight, eps=eps)
    if _any(outs):
        _native.check("mo_rotary_forward", lib.mo_rotary_forward(ctypes.byref(call), _stream(like)))
    return outs[0], outs[1]


def rotary_backward(grad_q: torch.Tensor | None, grad_k: torch.Tensor | None, table: torch.Tensor,
                    q: torch.Tensor | None = None, k: torch.Tensor | None = None, *, layout: str = "half",
                    q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                    eps: float = 1e-6) -> tuple[torch.Tensor | None, ...]:
    """``(d q, d k, d q_weight, d k_weight)`` from the outputs' gradients; ``q`` and ``k`` (the forward's inputs)
    are wanted where a weight is. What has no gradient is None."""

    lib = _native.load()
    call, _kept, outs, weight_grads, like = _call(((q, grad_q), (k, grad_k)), table, layout, (q_weight, k_weight), eps,
                                                  True)
    if _elsewhere(like):
        with torch.cuda.device(like.device):
            return rotary_backward(grad_q, grad_k, table, q, k, layout=layout, q_weight=q_weight, k_weight=k_weight,
                                   eps=eps)
    if _any(outs):
        nbytes = lib.mo_rotary_workspace_bytes(ctypes.byref(call)) if q_weight is not None or k_weight is not None else 0
        space = torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None
        _native.check("mo_rotary_backward", lib.mo_rotary_backward(
            ctypes.byref(call), 0 if space is None else space.data_ptr(), nbytes, _stream(like)))
    else:
        for grad in weight_grads:
            if grad is not None:
                grad.zero_()
    return outs[0], outs[1], weight_grads[0], weight_grads[1]


class _RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, table, q_weight, k_weight, layout, eps):
        ctx.layout, ctx.eps = layout, eps
        # without a norm the turn's gradient needs only the table
        ctx.save_for_backward(q if q_weight is not None else None, k if k_weight is not None else None, table, q_weight,
                              k_weight)
        return rotary_forward(q, k, table, layout=layout, q_weight=q_weight, k_weight=k_weight, eps=eps)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        q, k, table, q_weight, k_weight = ctx.saved_tensors
        grads = rotary_backward(grad_q, grad_k, table, q, k, layout=ctx.layout, q_weight=q_weight, k_weight=k_weight,
                                eps=ctx.eps)
        return grads[0], grads[1], None, grads[2], grads[3], None, None


def rotary(q: torch.Tensor | None, k: torch.Tensor | None, table: torch.Tensor, *, layout: str = "half",
           q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
           eps: float = 1e-6) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``rotary_forward`` with gradients for the queries, the keys and the norm weights; none for the table."""

    if table.requires_grad:
        raise RuntimeError("rotary has no gradient for its table.")
    return _RotaryFunction.apply(q, k, table, q_weight, k_weight, layout, eps)
