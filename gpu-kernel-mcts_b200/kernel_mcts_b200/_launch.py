"""Stream, device and argument handling shared by the expert-layer products.

A call costs about as long on the host as a small kernel runs, so each operand
is looked at once: :func:`rows_of` checks it and returns what the C call needs.
"""

from __future__ import annotations

import contextlib

import torch

MAX_GROUPS = 1024
MAX_SIZE = 2 ** 31 - 2 ** 10  # rows, N and K are 32-bit numbers in the kernels, with room to round up

_current_device = torch.cuda.current_device


def _refuse(name: str, tensor: torch.Tensor, dims: int, dtypes: tuple[torch.dtype, ...], index: int):
    if tensor.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}, got {tensor.dtype}")
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tensor.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}, got {tensor.device}")
    if tensor.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(tensor.shape)}")
    raise ValueError(f"{name} must be contiguous along its last dimension")


def row_stride(name: str, shape, strides, dim: int, unit: int) -> int:
    """Elements from one row to the next; where there is only one row, the
    row's length rounded up to `unit`, whatever stride torch reports."""
    length = shape[-1]
    if shape[dim] <= 1:
        return -(-length // unit) * unit
    stride = strides[dim]
    if stride < length:
        raise ValueError(f"{name} has overlapping rows (row stride {stride}, row length {length})")
    return stride


def rows_of(name: str, tensor: torch.Tensor, dims: int, dtypes: tuple[torch.dtype, ...], index: int, unit: int):
    """(shape, strides, row stride) of a tensor of one of the types on CUDA
    device `index` (negative, as get_device() of a CPU tensor, is refused), its
    innermost dimension contiguous."""
    shape = tensor.shape
    if tensor.dtype not in dtypes or len(shape) != dims or index < 0 or tensor.get_device() != index:
        _refuse(name, tensor, dims, dtypes, index)
    strides = tensor.stride()
    if shape[-1] > 1 and strides[-1] != 1:
        _refuse(name, tensor, dims, dtypes, index)
    return shape, strides, row_stride(name, shape, strides, -2, unit)


def check_groups(ends: torch.Tensor, index: int) -> int:
    if ends.dtype != torch.int32 or ends.dim() != 1 or not ends.is_contiguous():
        raise TypeError("ends must be a contiguous one-dimensional int32 tensor")
    if ends.get_device() != index:
        raise ValueError(f"ends must be on cuda:{index}, got {ends.device}")
    groups = ends.shape[0]
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"there must be 1 to {MAX_GROUPS} groups, got {groups}")
    return groups


def check_sizes(*sizes: int) -> None:
    if max(sizes) > MAX_SIZE:
        raise ValueError(f"sizes must be at most {MAX_SIZE}, got {sizes}")


def status_pointer(status: torch.Tensor | None, index: int) -> int | None:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.get_device() != index or status.numel() < 1:
        raise ValueError(f"status must be an int32 tensor on cuda:{index} with at least one element")
    return status.data_ptr()


class _Here:
    """The context of a call on the current device and stream: nothing to do."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return None


_HERE = _Here()


@contextlib.contextmanager
def _elsewhere(index: int, stream: torch.cuda.Stream | None):
    with torch.cuda.device(index):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def on_device(index: int, stream: torch.cuda.Stream | None):
    """The context a call allocates and launches in: the operands' device
    and the launching stream.  Results thus come from the memory of the stream
    that writes them, and cannot reuse a block that another stream's pending
    work still reads."""
    if stream is None:
        return _HERE if _current_device() == index else _elsewhere(index, None)
    if stream.device.index != index:
        raise ValueError(f"stream is on {stream.device}, the operands on cuda:{index}")
    return _elsewhere(index, stream)


def stream_handle(index: int) -> int:
    """The current stream's handle, inside :func:`on_device`."""
    return torch._C._cuda_getCurrentRawStream(index)


def caller_stream(index: int, stream: torch.cuda.Stream | None) -> torch.cuda.Stream | None:
    """The caller's stream when the call runs on another one, else None."""
    if stream is None:
        return None
    current = torch.cuda.current_stream(index)
    return current if current != stream else None


def use_on(stream: torch.cuda.Stream | None, caller: torch.cuda.Stream | None, *tensors: torch.Tensor | None) -> None:
    """Marks the caller's tensors as used by the side stream of a call, so
    that memory they free before the call is done waits for it."""
    if caller is not None:
        for tensor in tensors:
            if tensor is not None:
                tensor.record_stream(stream)


def share_result(result: torch.Tensor, caller: torch.cuda.Stream | None) -> torch.Tensor:
    """Marks a tensor allocated on a side stream as used by the stream the
    caller works on, so that its memory is not handed out again too early."""
    if caller is not None:
        result.record_stream(caller)
    return result
