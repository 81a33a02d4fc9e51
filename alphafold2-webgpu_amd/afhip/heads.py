"""What the operators over [batch][tokens][heads][channels] tensors share:
checks of tensors, and their strides for the C ABI."""
from __future__ import annotations

from . import _lib

FORMS = 64  # forms of a call (shapes, strides, types) an operator remembers


def form(tensor):
    """What a call's checks and descriptor depend on, of one tensor."""
    if tensor is None:
        return None
    return (tensor.shape, tensor.stride(), tensor.dtype, tensor.get_device())


def check_heads(name: str, tensor, dtype, shape, device: int, written: bool = False) -> None:
    """A device tensor [batch][tokens][heads][channels] of `dtype`, channels contiguous; `shape` may hold None."""
    check_device(name, tensor, device)
    if tensor.dtype != dtype:
        raise _lib.RangeError(f"{name} is {tensor.dtype}; this operator takes {dtype}")
    if tensor.dim() != 4 or any(want is not None and have != want for have, want in zip(tensor.shape, shape)):
        wanted = ", ".join("any" if want is None else str(want) for want in shape)
        raise _lib.RangeError(f"{name} has shape {tuple(tensor.shape)}; expected [{wanted}]")
    if tensor.stride(3) != 1 and tensor.shape[3] != 1:
        raise _lib.RangeError(f"{name} must have contiguous channels")
    if tensor.shape[1] > 1 and tensor.stride(1) == 0:
        raise _lib.RangeError(f"{name} repeats one token")
    if written and any(n > 1 and s == 0 for n, s in zip(tensor.shape, tensor.stride())):
        raise _lib.RangeError(f"{name} is written, and repeats one entry")


def check_ints(name: str, tensor, shape, device: int) -> None:
    import torch

    if tensor is None:
        return
    check_device(name, tensor, device)
    if tensor.dtype != torch.int32 or tuple(tensor.shape) != tuple(shape) or not tensor.is_contiguous():
        raise _lib.RangeError(f"{name} must be contiguous int32 of shape {tuple(shape)}")


def check_device(name: str, tensor, device: int) -> None:
    if tensor.get_device() != device or not tensor.is_cuda:
        raise _lib.RangeError(f"{name} is on {tensor.device}; afhip takes device tensors of cuda:{device}")


def strides(tensor) -> _lib.Strides:
    """A tensor's strides; an axis of one entry counts as packed."""
    _, tokens, heads, channels = tensor.shape
    head = tensor.stride(2) if heads > 1 else channels
    token = tensor.stride(1) if tokens > 1 else heads * channels
    batch = tensor.stride(0) if tensor.shape[0] > 1 else tokens * heads * channels
    return _lib.Strides(batch, token, head)


def address(tensor):
    return None if tensor is None else tensor.data_ptr()


def _direct(name: str, otherwise):
    """A getter of torch's own bindings where this torch has it, else the public one, which makes objects on the way
    (the current stream 2.7 us in place of 0.07, as long as the launch of a small kernel)."""
    import torch

    return getattr(torch._C, name, None) or otherwise(torch)


_stream = _device = None


def current_stream(index: int) -> int:
    """torch's current stream of a device, as a hipStream_t."""
    global _stream
    if _stream is None:
        _stream = _direct("_cuda_getCurrentRawStream",
                          lambda torch: lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _stream(index)


def current_device() -> int:
    global _device
    if _device is None:
        _device = _direct("_cuda_getDevice", lambda torch: torch.cuda.current_device)
    return _device()


def packed_like(tensor):
    """A new packed tensor of the same shape, type and device."""
    import torch

    return torch.empty_like(tensor, memory_format=torch.contiguous_format)
