"""What the calls on rows of activations (``norms``, ``gated``, ``adapters``, ``kept8``) check and look up alike."""

from __future__ import annotations

import torch

from . import _native
from .quant_kernels import _by_address

CODES = _native.DTYPE_CODES


def elsewhere(tensor: torch.Tensor, what: str) -> bool:
    """Whether the tensor's device is not the current one, which kernels are launched on."""

    index = tensor.get_device()
    if index < 0:
        raise RuntimeError(f"{what} operands must be on a HIP device.")
    return index != torch._C._cuda_getDevice()


def stream(tensor: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(tensor.get_device())


def plain(what: str, *operands: torch.Tensor | None) -> None:
    if not _by_address(*operands):
        raise RuntimeError(f"{what} operands must be plain tensors without a graph or a tangent; its autograd form has a "
                           "gradient.")


def rows(tensor: torch.Tensor, what: str) -> torch.Tensor:
    """``tensor`` as a matrix whose rows a kernel can read: dense, any distance apart."""

    if tensor.dtype not in CODES:
        raise TypeError(f"{what} must be bfloat16, float16 or float32 (got {tensor.dtype}).")
    if tensor.ndim == 0 or tensor.shape[-1] == 0:
        raise ValueError(f"{what} must have a last dimension, not empty.")
    cols = tensor.shape[-1]
    matrix = tensor if tensor.ndim == 2 else tensor.reshape(tensor.shape[:-1].numel(), cols)
    if (matrix.stride(1) != 1 and cols > 1) or (matrix.shape[0] > 1 and matrix.stride(0) < cols):
        matrix = matrix.contiguous()
    return matrix


def like(tensor: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """A contiguous tensor of ``tensor``'s shape, not filled: half the host time of ``torch.empty``."""

    return torch.empty_like(tensor, dtype=dtype, memory_format=torch.contiguous_format)


def pitch(matrix: torch.Tensor) -> int:
    return matrix.stride(0) if matrix.shape[0] > 1 else matrix.shape[1]


def whole(tensor: torch.Tensor | None, count: int, like: torch.Tensor, what: str) -> torch.Tensor | None:
    """A vector of ``count`` 64-bit whole numbers on ``like``'s device, as a kernel reads it."""

    if tensor is None:
        return None
    if tensor.dtype not in (torch.int64, torch.int32) or tensor.shape != (count,) \
            or tensor.get_device() != like.get_device():
        raise ValueError(f"{what} must be {count} int64 (or int32) numbers on the tokens' device.")
    return tensor if tensor.dtype == torch.int64 and tensor.is_contiguous() else tensor.to(torch.int64).contiguous()


def first_derivatives(what: str) -> None:
    """Called in a backward pass: what is kept for it carries no graph, so one that should build a graph is refused."""

    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no second derivatives (create_graph=True).")
