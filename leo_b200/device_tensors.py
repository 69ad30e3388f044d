"""What the operators on CUDA tensors share: element types, argument checks
and the stream that a call runs on."""

from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from .ctypes_types import BF16, F16, F32

DTYPE_CODES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}


def device_of(name: str, tensor) -> int:
    """The device index of a call's first tensor, which has to be a CUDA tensor."""
    index = tensor.get_device() if isinstance(tensor, torch.Tensor) else -1
    if index < 0 or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tensor.requires_grad or forward_ad._current_level >= 0:
        _refuse_gradient(name, tensor)
    return index


def dtype_code(name: str, tensor) -> int:
    code = DTYPE_CODES.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {tensor.dtype}")
    return code


def _refuse_gradient(name: str, tensor) -> None:
    if tensor.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient, which this call does not record: detach it and use the "
                         "gradients that the operators return")
    if forward_ad.unpack_dual(tensor).tangent is not None:
        raise ValueError(f"{name} has a tangent, which this call does not carry on")


def check_tensor(name: str, tensor, device: int, dtype=None, shape=None) -> None:
    """A tensor of the call: on CUDA device ``device``, asking for no gradient."""
    if (isinstance(tensor, torch.Tensor) and tensor.get_device() == device and (dtype is None or tensor.dtype == dtype)
            and (shape is None or tensor.shape == shape) and not tensor.requires_grad
            and forward_ad._current_level < 0):
        return
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tensor.get_device() != device:
        raise ValueError(f"{name} is on {tensor.device}, not on cuda:{device}")
    if dtype is not None and tensor.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {tensor.dtype}")
    if shape is not None and tensor.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(tensor.shape)}")
    _refuse_gradient(name, tensor)


def row_stride(name: str, tensor) -> int:
    """Elements between the rows of a 2-D tensor whose rows are adjacent elements."""
    if tensor.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, not {tensor.dim()}")
    stride = tensor.stride()
    if stride[1] != 1 and tensor.shape[1] > 1:
        raise ValueError(f"the elements of a row of {name} must be adjacent")
    return stride[0]


def check_contiguous(name: str, tensor) -> None:
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def pointer(tensor) -> int | None:
    return None if tensor is None else tensor.data_ptr()


def current_stream(device: int) -> int:
    """The raw current stream of a device."""
    return torch._C._cuda_getCurrentRawStream(device)


@contextlib.contextmanager
def _other_stream(stream, tensors):
    with torch.cuda.stream(stream):
        yield stream.cuda_stream
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


class _CurrentStream:
    """The raw current stream of a device, as a context that does nothing."""

    __slots__ = ("raw",)

    def __init__(self, raw: int):
        self.raw = raw

    def __enter__(self) -> int:
        return self.raw

    def __exit__(self, *exc) -> None:
        return None


def on_stream(device: int, stream, tensors):
    """The raw stream of a call: the current one of ``device``, or ``stream``.

    Outputs and scratch are to be allocated inside the context, so that they
    belong to the stream that writes them; with a ``stream`` other than the
    current one, ``tensors`` (the call's inputs) are marked as used on it."""
    if stream is None:
        return _CurrentStream(current_stream(device))
    if stream.device.index != device:
        raise ValueError(f"the stream is on {stream.device}, not on cuda:{device}")
    return _other_stream(stream, tensors)
