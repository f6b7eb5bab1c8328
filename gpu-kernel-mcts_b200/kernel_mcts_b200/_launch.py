"""Side streams for the expert-layer calls.

The calls themselves run on the operands' device and its current stream.
"""

from __future__ import annotations

import torch


def run_on(stream: torch.cuda.Stream, tensors, call, *args):
    """``call(*args)`` on ``stream``.

    Results come from the memory of the stream that writes them, so they cannot
    reuse a block that another stream's pending work still reads, and are marked
    as used by the caller's stream; the caller's tensors are marked as used by
    ``stream``.  Memory freed on either side before the work is done waits for it.
    """
    index = tensors[0].get_device()
    if index >= 0 and stream.device.index != index:
        raise ValueError(f"stream is on {stream.device}, the operands on cuda:{index}")
    caller = torch.cuda.current_stream(stream.device)
    if caller == stream:
        return call(*args)
    with torch.cuda.stream(stream):
        result = call(*args)
    for tensor in tensors:
        if tensor is not None:
            tensor.record_stream(stream)
    for tensor in result if isinstance(result, tuple) else (result,):
        tensor.record_stream(caller)
    return result
