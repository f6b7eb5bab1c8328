"""Microscaled 4-bit floating point (OCP MXFP4): quantisation and products.

An MXFP4 tensor of logical shape ``[..., K]`` is a pair of uint8 tensors:
``codes`` ``[..., K/2]``, two E2M1 codes a byte with the even element in the low
half, and ``scales`` ``[..., K/32]``, one E8M0 exponent (``2^(s - 127)``, 255 is
NaN) for each block of 32 elements.  Both may be views with strided rows, and
may be given as torch's ``float4_e2m1fn_x2`` and ``float8_e8m0fnu`` types.

The calls are not recorded by autograd: results require no gradient, and an
``out`` that requires one is refused while autograd records.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _launch, _native
from .grouped import kernel_code

BLOCK = 32

_calls = _native.torch_calls


class MXFP4Tensor(NamedTuple):
    """Packed codes and block scales; ``shape`` is the logical one."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], 2 * self.codes.shape[-1])


def mxfp4_quantize(
    x: torch.Tensor,
    out: MXFP4Tensor | None = None,
    *,
    stream: torch.cuda.Stream | None = None,
) -> MXFP4Tensor:
    """``x`` (bfloat16, float16 or float32, last dimension a multiple of 32)
    in MXFP4.

    The scale of a block is ``2^(floor(log2 m) - 2)`` for its largest magnitude
    ``m`` (at least ``2^-127``); elements round to the nearest code, ties to
    even, and saturate at 6 scales.  A block that holds an infinity or a NaN
    gets the NaN scale; its codes mean nothing.
    """
    codes, scales = out if out is not None else (None, None)
    if stream is None:
        return MXFP4Tensor(*_calls.mxfp4_quantize(x, codes, scales))
    return MXFP4Tensor(*_launch.run_on(stream, (x, codes, scales), _calls.mxfp4_quantize, x, codes, scales))


def mxfp4_dequantize(
    q: MXFP4Tensor,
    out: torch.Tensor | None = None,
    *,
    dtype: torch.dtype | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor:
    """The values of ``q`` in ``dtype`` (``out``'s type, or bfloat16), rounded
    once; exact in float32, and in bfloat16 from ``2^-133`` up."""
    if stream is None:
        return _calls.mxfp4_dequantize(*q, out, dtype)
    return _launch.run_on(stream, (*q, out), _calls.mxfp4_dequantize, *q, out, dtype)


def mxfp4_gemm(
    a: MXFP4Tensor,
    b: MXFP4Tensor,
    ends: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    *,
    kernel: str = "auto",
    stream: torch.cuda.Stream | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """``A·B^T`` of two MXFP4 operands: bfloat16 ``[rows, N]``, FP32 sums.

    ``a`` is ``[rows, K]``.  Without ``ends``, ``b`` is ``[N, K]``; with
    ``ends``, ``b`` is ``[groups, N, K]`` and each row of ``a`` meets its own
    group's weight; groups, ``out`` and ``kernel`` are as in
    :func:`kernel_mcts_b200.grouped.grouped_gemm`.  Code rows that do not start
    on 16 bytes take the CUDA-core kernel; scales may lie at any address.
    """
    args = (*a, *b, ends, out, kernel_code(kernel), status)
    if stream is None:
        return _calls.mxfp4_gemm(*args)
    return _launch.run_on(stream, (*a, *b, ends, out, status), _calls.mxfp4_gemm, *args)


__all__ = ["BLOCK", "MXFP4Tensor", "mxfp4_dequantize", "mxfp4_gemm", "mxfp4_quantize"]
