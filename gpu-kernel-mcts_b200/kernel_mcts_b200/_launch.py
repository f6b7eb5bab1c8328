"""Stream, device and argument handling shared by the expert-layer products."""

from __future__ import annotations

import contextlib

import torch

MAX_GROUPS = 1024


def check_tensor(name: str, tensor: torch.Tensor, dims: int, dtypes: tuple[torch.dtype, ...],
                 device: torch.device | None = None) -> None:
    """A CUDA tensor of one of the types, its innermost dimension contiguous."""
    if tensor.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}, got {tensor.dtype}")
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and tensor.device != device:
        raise ValueError(f"{name} must be on {device}, got {tensor.device}")
    if tensor.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(tensor.shape)}")
    if tensor.shape[-1] > 1 and tensor.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")


def row_stride(name: str, tensor: torch.Tensor, dim: int, unit: int) -> int:
    """Elements from one row to the next; where there is only one row, the
    row's length rounded up to `unit`, whatever stride torch reports."""
    length = tensor.shape[-1]
    if tensor.shape[dim] <= 1:
        return -(-length // unit) * unit
    stride = tensor.stride(dim)
    if stride < length:
        raise ValueError(f"{name} has overlapping rows (row stride {stride}, row length {length})")
    return stride


def check_groups(ends: torch.Tensor, device: torch.device) -> int:
    if ends.dtype != torch.int32 or ends.dim() != 1 or not ends.is_contiguous():
        raise TypeError("ends must be a contiguous one-dimensional int32 tensor")
    if ends.device != device:
        raise ValueError(f"ends must be on {device}, got {ends.device}")
    groups = ends.shape[0]
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"there must be 1 to {MAX_GROUPS} groups, got {groups}")
    return groups


def status_pointer(status: torch.Tensor | None, device: torch.device) -> int | None:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.device != device or status.numel() < 1:
        raise ValueError(f"status must be an int32 tensor on {device} with at least one element")
    return status.data_ptr()


@contextlib.contextmanager
def _on(device: torch.device, stream: torch.cuda.Stream | None):
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def on_device(device: torch.device, stream: torch.cuda.Stream | None):
    """The context a call allocates and launches in: the operands' device
    and the launching stream.  Results thus come from the memory of the stream
    that writes them, and cannot reuse a block that another stream's pending
    work still reads."""
    if stream is None and torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    if stream is not None and stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the operands on {device}")
    return _on(device, stream)


def stream_handle(device: torch.device, stream: torch.cuda.Stream | None) -> int:
    return (stream if stream is not None else torch.cuda.current_stream(device)).cuda_stream


def share_result(result: torch.Tensor, caller: torch.cuda.Stream | None) -> None:
    """Marks a tensor allocated on a side stream as used by the stream the
    caller works on, so that its memory is not handed out again too early."""
    if caller is not None:
        result.record_stream(caller)


def caller_stream(device: torch.device, stream: torch.cuda.Stream | None) -> torch.cuda.Stream | None:
    """The caller's stream when the call runs on another one, else None."""
    if stream is None:
        return None
    current = torch.cuda.current_stream(device)
    return current if current != stream else None
