"""Linears in 8-bit floating point on the f8f6f4 matrix cores, with a scale for each 128 values.

A matrix is kept as e4m3 bytes and one scale a group: 128 values along a row (``fp8_quantize_rows``), 128
along a column (``fp8_quantize_columns``), or a 128 x 128 block of a weight (``fp8_quantize_weight``).
The scales made here are powers of two (``float8_e8m0fnu``, one byte): the smallest, from 2**-126 on,
that brings the group within e4m3's largest value, 448. The matrix instructions apply them, so a product
needs no arithmetic for its scales. Weights from elsewhere may carry any float32 block scales.

Three products share them (``csrc/mo_fp8.hip``), fp32 sums, each rounded once to its output type:

- ``fp8_linear_forward``: ``Q(tokens) @ W.T (+ bias)``, tokens quantized along their rows;
- ``fp8_linear_backward``: ``Q(gradient) @ W``, the gradient quantized along its rows;
- ``fp8_weight_gradient``: ``Q(gradient).T @ Q(tokens)``, both quantized along the tokens.

``fp8_linear`` puts them under autograd, for a frozen weight or for one in training (first derivatives; a
backward that should build a graph through a weight in training raises). The reference has no
floating-point 8-bit base; its int8 one (``training/quantization.py:23-131``) is ``quant_kernels`` here.

Feature sizes are multiples of 16, rows any number. A group with an infinity or a NaN reads back as NaN.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _native
from .quant_kernels import _by_address

GROUP = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LARGEST = 448.0
_CODES = _native.DTYPE_CODES


def _elsewhere(tensor: torch.Tensor) -> bool:
    """Whether the tensor's device is not the current one, which kernels are launched on."""

    index = tensor.get_device()
    if index < 0:
        raise RuntimeError("fp8 operands must be on a HIP device.")
    return index != torch._C._cuda_getDevice()


def _stream(tensor: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(tensor.get_device())


def _groups(size: int) -> int:
    return -(-size // GROUP)


def _scales(rows: int, size: int, device) -> torch.Tensor:
    """Room for one scale for each 128 of ``size`` values of ``rows`` rows: ``[rows, groups]``, laid group by
    group (what the products read at a time is then dense)."""

    groups, pitch = -(-size // GROUP), -(-rows // 16) * 16
    return torch.empty(groups * pitch, dtype=E8M0, device=device).as_strided((rows, groups), (1, pitch))


def _plain(*operands: torch.Tensor | None) -> None:
    if not _by_address(*operands):
        raise RuntimeError("fp8 operands must be plain tensors without a graph or a tangent; fp8_linear has a gradient "
                           "(none for a block-scaled weight or its scales).")


def _rows(tensor: torch.Tensor, what: str) -> torch.Tensor:
    """``tensor`` as a matrix whose rows a kernel can read: dense, 16-byte aligned, any distance apart."""

    if tensor.dtype not in _CODES:
        raise TypeError(f"fp8 {what} must be bfloat16, float16 or float32 (got {tensor.dtype}).")
    if tensor.ndim == 0 or tensor.shape[-1] == 0 or tensor.shape[-1] % 16:
        raise ValueError(f"fp8 {what} must have a last dimension that is a multiple of 16.")
    matrix = tensor if tensor.ndim == 2 else tensor.reshape(-1, tensor.shape[-1])
    rows, cols = matrix.shape
    unit = 16 // matrix.element_size()
    if matrix.stride(1) != 1 or (rows > 1 and (matrix.stride(0) < cols or matrix.stride(0) % unit)):
        matrix = matrix.contiguous()
    return matrix.clone() if matrix.data_ptr() % 16 else matrix


def _stride(matrix: torch.Tensor) -> int:
    return matrix.stride(0) if matrix.shape[0] > 1 else matrix.shape[1]


def _weight(weight: torch.Tensor, scale: torch.Tensor) -> int:
    """The scale kind of a block-scaled weight, after its checks: every kernel takes it by address."""

    _plain(weight, scale)
    if weight.ndim != 2 or weight.dtype != E4M3 or not weight.is_contiguous() or weight.data_ptr() % 16:
        raise RuntimeError("fp8 weight must be a contiguous, 16-byte aligned float8_e4m3fn matrix.")
    if weight.shape[0] % 16 or weight.shape[1] % 16 or not weight.numel():
        raise RuntimeError("fp8 weight must have features that are multiples of 16.")
    if scale.dtype not in (E8M0, torch.float32) or scale.shape != (_groups(weight.shape[0]), _groups(weight.shape[1])) \
            or not scale.is_contiguous() or scale.get_device() != weight.get_device():
        raise RuntimeError("fp8 weight scale must be contiguous float8_e8m0fnu or float32 on the weight's device, "
                           "one for each block of 128 x 128.")
    return _native.MO_FP8_SCALE_F32 if scale.dtype == torch.float32 else _native.MO_FP8_SCALE_E8M0


def _pair(pair: tuple[torch.Tensor, torch.Tensor], features: int, what: str) -> tuple[torch.Tensor, torch.Tensor]:
    """A quantized operand as the kernels read it: dense rows, scales group by group."""

    values, scales = pair
    if values.dtype != E4M3 or scales.dtype != E8M0 or values.ndim < 1 or values.shape[-1] != features:
        raise RuntimeError(f"quantized fp8 {what} must be float8_e4m3fn of {features} features with float8_e8m0fnu scales.")
    rows, groups = values.shape[:-1].numel(), _groups(features)
    values = values.reshape(rows, features).contiguous()  # the rows of no tokens hold nothing: -1 would be ambiguous
    if values.data_ptr() % 16:
        values = values.clone()
    if scales.shape != (rows, groups) or scales.get_device() != values.get_device():
        raise RuntimeError(f"quantized fp8 {what} must have one scale for each 128 values of a row, on its device.")
    if rows and (scales.stride(0) != 1 or groups > 1 and scales.stride(1) != -(-rows // 16) * 16
                 or scales.data_ptr() % 4
                 # a row's end is read in whole words
                 or scales.untyped_storage().nbytes() - scales.storage_offset() < groups * (-(-rows // 16) * 16)):
        laid = _scales(rows, features, scales.device)
        laid.view(torch.uint8).copy_(scales.view(torch.uint8))
        scales = laid
    return values, scales


def _output(out: torch.Tensor | None, shape: tuple[int, int], dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if dtype not in _CODES:
        raise TypeError(f"fp8 output must be bfloat16, float16 or float32 (got {dtype}).")
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _plain(out)
    if out.dtype != dtype or not out.is_contiguous() or out.numel() != shape[0] * shape[1] or out.device != device \
            or out.data_ptr() % 16:
        raise ValueError("fp8 output buffer has the wrong dtype, size or device, or is not contiguous and aligned.")
    return out.view(shape)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(op: int, rows: int, in_features: int, out_features: int, quantized: bool, kind: int, code: int,
                     device: int) -> int:
    lib = _native.load()
    nbytes = lib.mo_fp8_workspace_bytes(op, rows, in_features, out_features, int(quantized), kind, code)
    if nbytes == _native.MO_FP8_NO_SIZE:  # an exception is not cached: the next call asks again
        raise _native.EngineError("mo_fp8_workspace_bytes", -1, lib.mo_last_error().decode(errors="replace"))
    return nbytes


def _workspace(op: int, rows: int, in_features: int, out_features: int, quantized: bool, kind: int, dtype: torch.dtype,
               like: torch.Tensor) -> tuple:
    # freed to the caching allocator after the call; stream order keeps it alive for the kernels
    nbytes = _workspace_bytes(op, rows, in_features, out_features, quantized, kind, _CODES[dtype], like.get_device())
    return (torch.empty(nbytes, dtype=torch.uint8, device=like.device), nbytes) if nbytes else (None, 0)


def _address(tensor: torch.Tensor | None) -> int:
    return 0 if tensor is None else tensor.data_ptr()


# ---- quantizing and reading back ------------------------------------------------------------------


def _quantize(x: torch.Tensor, rows: bool, columns: bool):
    lib = _native.load()
    _plain(x)
    matrix = _rows(x, "matrix")
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return _quantize(x, rows, columns)
    (m, n), device = matrix.shape, x.device
    row = column = None
    pointers = [0, 0, 0, 0]
    if rows:
        row = torch.empty(x.shape, dtype=E4M3, device=device), _scales(m, n, device)
        pointers[:2] = row[0].data_ptr(), row[1].data_ptr()
    if columns:
        column = torch.empty((n, -(-m // GROUP) * GROUP), dtype=E4M3, device=device), _scales(n, m, device)
        pointers[2:] = column[0].data_ptr(), column[1].data_ptr()
    if m:
        _native.check("mo_fp8_quantize", lib.mo_fp8_quantize(
            matrix.data_ptr(), _CODES[matrix.dtype], m, n, _stride(matrix), *pointers, _stream(x)))
    return row, column


def fp8_quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, scales)`` of a matrix (or rows of any leading shape, or one row) in groups of 128 along its
    rows: values of ``x``'s shape, one scale ``[rows, ceil(cols / 128)]``."""

    return _quantize(x, True, False)[0]


def fp8_quantize_columns(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, scales)`` of ``x`` transposed, in groups of 128 along its columns: values ``[cols, rows
    rounded up to 128]`` (the end zero), scales ``[cols, ceil(rows / 128)]``."""

    return _quantize(x, False, True)[1]


def fp8_quantize_both(x: torch.Tensor) -> tuple[tuple[torch.Tensor, torch.Tensor], tuple[torch.Tensor, torch.Tensor]]:
    """``(fp8_quantize_rows(x), fp8_quantize_columns(x))`` in one reading of ``x``."""

    return _quantize(x, True, True)


def fp8_quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, scales)`` of a weight ``[out, in]`` in blocks of 128 x 128. (``out`` is any number here; the
    products take multiples of 16.)"""

    lib = _native.load()
    _plain(weight)
    if weight.ndim != 2 or not weight.shape[0]:
        raise ValueError("fp8 weight must be a matrix, not empty.")
    matrix = _rows(weight, "weight")
    if _elsewhere(weight):
        with torch.cuda.device(weight.device):
            return fp8_quantize_weight(weight)
    rows, cols = matrix.shape
    values = torch.empty((rows, cols), dtype=E4M3, device=weight.device)
    scales = torch.empty((_groups(rows), _groups(cols)), dtype=E8M0, device=weight.device)
    _native.check("mo_fp8_quantize_weight", lib.mo_fp8_quantize_weight(
        matrix.data_ptr(), _CODES[matrix.dtype], rows, cols, _stride(matrix), values.data_ptr(), scales.data_ptr(),
        _stream(weight)))
    return values, scales


def fp8_decode(values: torch.Tensor, scales: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16,
               cols: int | None = None) -> torch.Tensor:
    """The matrix that ``(values, scales)`` stand for, in ``dtype``: one scale for each 128 values of a row,
    or of a block of 128 x 128, as ``scales``'s rows say. ``cols``: of each row, as many values."""

    lib = _native.load()
    _plain(values, scales)
    if values.dtype != E4M3 or values.ndim < 1 or scales.dtype not in (E8M0, torch.float32) or scales.ndim != 2:
        raise TypeError("fp8_decode takes float8_e4m3fn values with float8_e8m0fnu or float32 scales.")
    if dtype not in _CODES:
        raise TypeError(f"fp8 output must be bfloat16, float16 or float32 (got {dtype}).")
    if values.shape[-1] == 0 or values.shape[-1] % 16:
        raise ValueError("fp8 values must have a last dimension that is a multiple of 16.")
    matrix = values if values.ndim == 2 else values.reshape(-1, values.shape[-1])
    cols = matrix.shape[1] if cols is None else cols
    if not 0 <= cols <= matrix.shape[1]:
        raise ValueError("fp8_decode's cols must lie within the values.")
    rows = matrix.shape[0]
    if matrix.stride(1) != 1 or (rows > 1 and (matrix.stride(0) < matrix.shape[1] or matrix.stride(0) % 16)) \
            or matrix.data_ptr() % 16:
        matrix = matrix.contiguous()
        matrix = matrix.clone() if matrix.data_ptr() % 16 else matrix
    if scales.shape[0] not in (rows, _groups(rows)) or scales.shape[1] < _groups(cols) \
            or scales.get_device() != values.get_device():
        raise ValueError("fp8 scales do not fit the values.")
    if _elsewhere(values):
        with torch.cuda.device(values.device):
            return fp8_decode(values, scales, dtype=dtype, cols=cols)
    out = torch.empty((*values.shape[:-1], cols), dtype=dtype, device=values.device)
    if rows and cols:
        kind = _native.MO_FP8_SCALE_F32 if scales.dtype == torch.float32 else _native.MO_FP8_SCALE_E8M0
        _native.check("mo_fp8_decode", lib.mo_fp8_decode(
            matrix.data_ptr(), _stride(matrix), scales.data_ptr(), kind, scales.stride(0), scales.stride(1),
            1 if scales.shape[0] == rows else GROUP, out.data_ptr(), _CODES[dtype], rows, cols, _stream(values)))
    return out


# ---- products -------------------------------------------------------------------------------------


def _operand(given, features: int, what: str):
    """(values or matrix, scales or None, its type's code, rows, stride, leading shape) of a product's operand."""

    if isinstance(given, (tuple, list)):
        values, scales = _pair(given, features, what)
        _plain(values, scales)
        return values, scales, 0, values.shape[0], features, given[0].shape[:-1]
    _plain(given)
    matrix = _rows(given, what)
    if matrix.shape[1] != features:
        raise ValueError(f"fp8 {what} must have {features} features (got {matrix.shape[1]}).")
    return matrix, None, _CODES[matrix.dtype], matrix.shape[0], _stride(matrix), given.shape[:-1]


def fp8_linear_forward(tokens, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None, *,
                       dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``Q(tokens) @ decode(weight, scale).T (+ bias)``. ``tokens``: ``[..., in]``, quantized along its rows,
    or the pair that ``fp8_quantize_rows`` gives. ``weight``: e4m3 ``[out, in]``; ``scale``: one for each
    128 x 128 block, e8m0 or float32. ``bias``: ``[out]`` of any floating type, added to the float32 sum. ``dtype``:
    the result's (the tokens' own; bfloat16 for a pair). The result has no graph: ``fp8_linear`` has one."""

    lib = _native.load()
    kind = _weight(weight, scale)
    out_features, in_features = weight.shape
    matrix, scales, code, rows, stride, lead = _operand(tokens, in_features, "tokens")
    if matrix.get_device() != weight.get_device():
        raise RuntimeError("fp8 tokens and weight must be on one device.")
    if _elsewhere(weight):
        with torch.cuda.device(weight.device):
            return fp8_linear_forward(tokens, weight, scale, bias, dtype=dtype, out=out)
    dtype = dtype or (torch.bfloat16 if scales is not None else matrix.dtype)
    result = _output(out, (rows, out_features), dtype, weight.device)
    kinds = _CODES[dtype]
    if bias is not None:
        _plain(bias)
        if bias.shape != (out_features,) or bias.get_device() != weight.get_device():
            raise RuntimeError(f"fp8 bias must be {out_features} values on the weight's device.")
        # added in fp32, before the one rounding: another type than the result's goes in as float32
        bias = (bias if bias.dtype == dtype else bias.float()).contiguous()
        kinds |= _native.MO_FP8_BIAS_F32 if bias.dtype == torch.float32 else 0
    if rows:
        space, nbytes = _workspace(_native.MO_FP8_FORWARD, rows, in_features, out_features, scales is not None, kind,
                                   dtype, weight)
        _native.check("mo_fp8_linear_forward", lib.mo_fp8_linear_forward(
            matrix.data_ptr(), _address(scales), code, rows, in_features, stride, weight.data_ptr(), scale.data_ptr(),
            kind, out_features, _address(bias), result.data_ptr(), kinds, _address(space), nbytes, _stream(weight)))
    return result if len(lead) == 1 else result.view(*lead, out_features)


def fp8_linear_backward(gradient, weight: torch.Tensor, scale: torch.Tensor, *, dtype: torch.dtype | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``Q(gradient) @ decode(weight, scale)``: the input gradient. ``gradient``: ``[..., out]``, quantized
    along its rows, or the pair that ``fp8_quantize_rows`` gives; the rest as in ``fp8_linear_forward``."""

    lib = _native.load()
    kind = _weight(weight, scale)
    out_features, in_features = weight.shape
    matrix, scales, code, rows, stride, lead = _operand(gradient, out_features, "gradient")
    if matrix.get_device() != weight.get_device():
        raise RuntimeError("fp8 gradient and weight must be on one device.")
    if _elsewhere(weight):
        with torch.cuda.device(weight.device):
            return fp8_linear_backward(gradient, weight, scale, dtype=dtype, out=out)
    dtype = dtype or (torch.bfloat16 if scales is not None else matrix.dtype)
    result = _output(out, (rows, in_features), dtype, weight.device)
    if rows:
        space, nbytes = _workspace(_native.MO_FP8_BACKWARD, rows, in_features, out_features, scales is not None, kind,
                                   dtype, weight)
        _native.check("mo_fp8_linear_backward", lib.mo_fp8_linear_backward(
            matrix.data_ptr(), _address(scales), code, rows, in_features, out_features, stride, weight.data_ptr(),
            scale.data_ptr(), kind, result.data_ptr(), _CODES[dtype], _address(space), nbytes, _stream(weight)))
    return result if len(lead) == 1 else result.view(*lead, in_features)


def fp8_weight_gradient(gradient, tokens, *, rows: int | None = None, dtype: torch.dtype = torch.float32,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``Q(gradient).T @ Q(tokens)``, ``[out, in]`` in ``dtype``: the weight gradient. ``gradient``: ``[..., out]``
    and ``tokens``: ``[..., in]``, both quantized along their rows' direction in groups of 128 tokens, or
    the pairs that ``fp8_quantize_columns`` gives for them (then ``rows``: the tokens)."""

    lib = _native.load()
    quantized = isinstance(gradient, (tuple, list))
    if quantized != isinstance(tokens, (tuple, list)):
        raise TypeError("fp8_weight_gradient takes two matrices or two quantized pairs.")
    if quantized:
        if rows is None:
            raise ValueError("fp8_weight_gradient needs the number of tokens of quantized pairs.")
        padded = _groups(rows) * GROUP
        dy, dy_scales = _pair(gradient, padded, "gradient")
        x, x_scales = _pair(tokens, padded, "tokens")
        _plain(dy, dy_scales, x, x_scales)
        out_features, in_features = dy.shape[0], x.shape[0]
        dy_code = x_code = 0
        dy_stride = x_stride = padded
        if out_features % 16 or in_features % 16 or not out_features or not in_features:
            raise ValueError("fp8_weight_gradient takes features that are multiples of 16.")
    else:
        _plain(gradient, tokens)
        dy, x, dy_scales, x_scales = _rows(gradient, "gradient"), _rows(tokens, "tokens"), None, None
        if gradient.shape[:-1] != tokens.shape[:-1] or rows not in (None, dy.shape[0]):
            raise ValueError("fp8 gradient and tokens must have the same rows.")
        rows, out_features, in_features = dy.shape[0], dy.shape[1], x.shape[1]
        dy_code, x_code, dy_stride, x_stride = _CODES[dy.dtype], _CODES[x.dtype], _stride(dy), _stride(x)
    if dy.get_device() != x.get_device():
        raise RuntimeError("fp8 gradient and tokens must be on one device.")
    if _elsewhere(dy):
        with torch.cuda.device(dy.device):
            return fp8_weight_gradient(gradient, tokens, rows=rows, dtype=dtype, out=out)
    result = _output(out, (out_features, in_features), dtype, dy.device)
    if not rows:
        return result.zero_()
    space, nbytes = _workspace(_native.MO_FP8_WEIGHT, rows, in_features, out_features, quantized,
                               _native.MO_FP8_SCALE_E8M0, dtype, dy)
    _native.check("mo_fp8_weight_gradient", lib.mo_fp8_weight_gradient(
        dy.data_ptr(), _address(dy_scales), dy_code, dy_stride, x.data_ptr(), _address(x_scales), x_code, x_stride,
        rows, in_features, out_features, result.data_ptr(), _CODES[dtype], _address(space), nbytes, _stream(dy)))
    return result


def product_plan(rows: int, cols: int, reduction: int, cus: int, *, float_scales: bool = False,
                 dtype: torch.dtype = torch.bfloat16) -> list[dict]:
    """How a product ``[rows, cols]`` from a ``reduction`` runs on a device of ``cus`` CUs (``mo_fp8_plan``):
    one or two launches, each ``{"rows", "edge"}`` of its tile, ``"splits"`` of the reduction and
    ``"split_steps"`` of 128 each."""

    raw = (ctypes.c_uint32 * 8)()
    kind = _native.MO_FP8_SCALE_F32 if float_scales else _native.MO_FP8_SCALE_E8M0
    _native.check("mo_fp8_plan", _native.load().mo_fp8_plan(rows, cols, reduction, kind, _CODES[dtype], cus, raw))
    return [dict(zip(("rows", "edge", "splits", "split_steps"), raw[4 * i : 4 * i + 4])) for i in range(2) if raw[4 * i]]


# ---- under autograd -------------------------------------------------------------------------------


def _bias_gradient(gradient: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return gradient.reshape(-1, gradient.shape[-1]).sum(0, dtype=torch.float32).to(dtype)


class _FrozenFunction(torch.autograd.Function):
    """A frozen weight: saves the weight and its scales, which are the module's own buffers."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, bias, dtype):
        ctx.save_for_backward(weight, scale)
        ctx.input_dtype = tokens.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return fp8_linear_forward(tokens, weight, scale, bias, dtype=dtype)

    @staticmethod
    def backward(ctx, gradient):
        weight, scale = ctx.saved_tensors
        wanted, bias_wanted = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
        tokens = fp8_linear_backward(gradient, weight, scale, dtype=ctx.input_dtype) if wanted else None
        bias = _bias_gradient(gradient, ctx.bias_dtype) if bias_wanted else None
        return tokens, None, None, bias, None


class _TrainedFunction(torch.autograd.Function):
    """A weight in training: quantized for the call; the tokens are kept in 8 bits, turned for the weight
    gradient (half the bytes that a bfloat16 linear keeps), and the weight's 8 bits for the input gradient.
    What is kept carries no graph, while the tokens' gradient depends on the weight and the weight's on the
    tokens: where both are wanted, a backward that should build a graph is refused."""

    @staticmethod
    def forward(ctx, tokens, weight, bias, dtype, graph):
        values, scale = fp8_quantize_weight(weight)
        if not graph:  # needs_input_grad is set all the same
            return fp8_linear_forward(tokens, values, scale, bias, dtype=dtype)
        ctx.input_dtype, ctx.weight_dtype = tokens.dtype, weight.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.rows = tokens.shape[:-1].numel()
        ctx.both = ctx.needs_input_grad[0] and ctx.needs_input_grad[1]
        if ctx.needs_input_grad[1]:
            tokens, columns = fp8_quantize_both(tokens)
        else:
            columns = (None, None)
        ctx.save_for_backward(values, scale, *columns)
        return fp8_linear_forward(tokens, values, scale, bias, dtype=dtype)

    @staticmethod
    def backward(ctx, gradient):
        if ctx.both and torch.is_grad_enabled():
            raise RuntimeError("fp8_linear has no second derivatives for a weight in training (create_graph=True).")
        values, scale, *columns = ctx.saved_tensors
        tokens = weight = bias = None
        if ctx.needs_input_grad[2]:
            bias = _bias_gradient(gradient, ctx.bias_dtype)
        rows, turned = gradient, None
        if ctx.needs_input_grad[0] and ctx.needs_input_grad[1]:
            rows, turned = fp8_quantize_both(gradient)
        elif ctx.needs_input_grad[1]:
            turned = fp8_quantize_columns(gradient)
        if ctx.needs_input_grad[0]:
            tokens = fp8_linear_backward(rows, values, scale, dtype=ctx.input_dtype)
        if ctx.needs_input_grad[1]:
            weight = fp8_weight_gradient(turned, tuple(columns), rows=ctx.rows, dtype=ctx.weight_dtype)
        return tokens, weight, bias, None, None


def fp8_linear(tokens: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """A linear in 8-bit floating point with its gradients. With ``scale``: a frozen block-scaled weight; one that
    wants a gradient, or whose scales do, is refused.
    Without: ``weight`` is ``[out, in]`` in bfloat16, float16 or float32, quantized for the call, and gets
    a gradient of its own type. ``dtype``: the result's (the tokens' own)."""

    dtype = dtype or tokens.dtype
    if scale is not None:
        _plain(weight, scale)  # seen here: inside the function grad mode is off
        return _FrozenFunction.apply(tokens, weight, scale, bias, dtype)
    return _TrainedFunction.apply(tokens, weight, bias, dtype, torch.is_grad_enabled())
