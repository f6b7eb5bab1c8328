"""Microscaled 4-bit floating point (OCP MXFP4): quantisation and products.

An MXFP4 tensor of logical shape ``[..., K]`` is a pair of uint8 tensors:
``codes`` ``[..., K/2]``, two E2M1 codes a byte with the even element in the low
half, and ``scales`` ``[..., K/32]``, one E8M0 exponent (``2^(s - 127)``, 255 is
NaN) for each block of 32 elements.  Both may be views with strided rows, and
may be given as torch's ``float4_e2m1fn_x2`` and ``float8_e8m0fnu`` types.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _launch, _native
from .grouped import kernel_code

BLOCK = 32

_TYPES = {
    torch.bfloat16: _native.TYPE_BF16,
    torch.float16: _native.TYPE_FP16,
    torch.float32: _native.TYPE_FP32,
}
_TYPE_TUPLE = tuple(_TYPES)
_BF16 = (torch.bfloat16,)
_CODES = (torch.uint8, torch.float4_e2m1fn_x2)
_SCALES = (torch.uint8, torch.float8_e8m0fnu)


class MXFP4Tensor(NamedTuple):
    """Packed codes and block scales; ``shape`` is the logical one."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], 2 * self.codes.shape[-1])


def _pair_rows(name: str, q: MXFP4Tensor, dims: int, index: int):
    """(code shape, code strides, code row stride, scale strides, scale row
    stride) of a checked pair."""
    shape, strides, ldc = _launch.rows_of(f"{name} codes", q[0], dims, _CODES, index, 16)
    scale_shape, scale_strides, lds = _launch.rows_of(f"{name} scales", q[1], dims, _SCALES, index, 1)
    if shape[-1] % (BLOCK // 2) != 0:
        raise ValueError(f"{name} has K={2 * shape[-1]}, not a multiple of {BLOCK}")
    if scale_shape[-1] != shape[-1] // (BLOCK // 2) or scale_shape[:-1] != shape[:-1]:
        want = (*shape[:-1], shape[-1] // (BLOCK // 2))
        raise ValueError(f"{name} scales must have shape {want}, got {tuple(scale_shape)}")
    return shape, strides, ldc, scale_strides, lds


def _rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """The tensor as rows of its last dimension."""
    if t.dim() == 2:
        return t
    if t.dim() < 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be two-dimensional or contiguous")
    return t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])


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
    shape = x.shape
    if len(shape) < 1 or shape[-1] % BLOCK != 0:
        raise ValueError(f"x must have a last dimension that is a multiple of {BLOCK}, got shape {tuple(shape)}")
    flat = _rows("x", x)
    device = x.get_device()
    (rows, k), _, ldx = _launch.rows_of("x", flat, 2, _TYPE_TUPLE, device, BLOCK)
    _launch.check_sizes(k)
    caller = _launch.caller_stream(device, stream)
    _launch.use_on(stream, caller, x, *(out or ()))
    with _launch.on_device(device, stream):
        if out is None:
            lead = shape[:-1]
            codes = _launch.share_result(x.new_empty((*lead, k // 2), dtype=torch.uint8), caller)
            scales = _launch.share_result(x.new_empty((*lead, k // BLOCK), dtype=torch.uint8), caller)
            out, ldc, lds = MXFP4Tensor(codes, scales), k // 2, k // BLOCK
        else:
            codes, scales = _rows("out codes", out.codes), _rows("out scales", out.scales)
            _, _, ldc, _, lds = _pair_rows("out", MXFP4Tensor(codes, scales), 2, device)
            if out.shape != tuple(shape):
                raise ValueError(f"out must have shape {tuple(shape)}, got {out.shape}")
        rc = _native.load().kmcts_mxfp4_quantize(
            flat.data_ptr(), _TYPES[x.dtype], ldx, codes.data_ptr(), ldc, scales.data_ptr(), lds, rows, k,
            _launch.stream_handle(device))
    if rc:
        _native.check(rc, "kmcts_mxfp4_quantize")
    return out


def mxfp4_dequantize(
    q: MXFP4Tensor,
    out: torch.Tensor | None = None,
    *,
    dtype: torch.dtype | None = None,
    stream: torch.cuda.Stream | None = None,
) -> torch.Tensor:
    """The values of ``q`` in ``dtype`` (``out``'s type, or bfloat16), rounded
    once; exact in float32, and in bfloat16 from ``2^-133`` up."""
    codes, scales = _rows("q codes", q[0]), _rows("q scales", q[1])
    device = codes.get_device()
    (rows, half), _, ldc, _, lds = _pair_rows("q", MXFP4Tensor(codes, scales), 2, device)
    if q.scales.shape[:-1] != q.codes.shape[:-1]:
        raise ValueError(f"q scales must go with codes of shape {tuple(q.codes.shape)}, got {tuple(q.scales.shape)}")
    k = 2 * half
    _launch.check_sizes(k)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16
    if dtype not in _TYPES:
        raise TypeError(f"values must be bfloat16, float16 or float32, got {dtype}")
    caller = _launch.caller_stream(device, stream)
    _launch.use_on(stream, caller, *q, out)
    with _launch.on_device(device, stream):
        if out is None:
            flat = out = _launch.share_result(codes.new_empty(q.shape, dtype=dtype), caller)
            ldo = k
        else:
            if tuple(out.shape) != q.shape:
                raise ValueError(f"out must have shape {q.shape}, got {tuple(out.shape)}")
            flat = _rows("out", out)
            _, _, ldo = _launch.rows_of("out", flat, 2, (dtype,), device, BLOCK)
        rc = _native.load().kmcts_mxfp4_dequantize(
            codes.data_ptr(), ldc, scales.data_ptr(), lds, flat.data_ptr(), _TYPES[dtype], ldo, rows, k,
            _launch.stream_handle(device))
    if rc:
        _native.check(rc, "kmcts_mxfp4_dequantize")
    return out


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
    device = a[0].get_device()
    (rows, half), _, lda, _, ldas = _pair_rows("a", a, 2, device)
    b_shape, b_strides, ldb, bs_strides, ldbs = _pair_rows("b", b, 2 if ends is None else 3, device)
    if b_shape[-1] != half:
        raise ValueError(f"inner dimensions differ: a has K={2 * half}, b has K={2 * b_shape[-1]}")
    k, n = 2 * half, b_shape[-2]
    _launch.check_sizes(rows, n, k)
    groups, ends_ptr, b_stride, bs_stride = 1, None, 0, 0
    if ends is not None:
        groups, ends_ptr = _launch.check_groups(ends, device), ends.data_ptr()
        if b_shape[0] != groups:
            raise ValueError(f"b holds {b_shape[0]} groups, ends {groups}")
        if groups > 1:
            b_stride, bs_stride = b_strides[0], bs_strides[0]
    status_ptr = _launch.status_pointer(status, device)
    kernel_id = kernel_code(kernel)
    caller = _launch.caller_stream(device, stream)
    _launch.use_on(stream, caller, *a, *b, ends, out, status)
    with _launch.on_device(device, stream):
        if out is None:
            out = _launch.share_result(a[1].new_empty((rows, n), dtype=torch.bfloat16), caller)
            ldy, flags = n, _native.GROUPED_ZERO_REST
        else:
            shape, _, ldy = _launch.rows_of("out", out, 2, _BF16, device, 8)
            if shape != (rows, n):
                raise ValueError(f"out must have shape {(rows, n)}, got {tuple(shape)}")
            flags = 0
        rc = _native.load().kmcts_mxfp4_gemm(
            a[0].data_ptr(), lda, a[1].data_ptr(), ldas, b[0].data_ptr(), b_stride, ldb, b[1].data_ptr(), bs_stride, ldbs,
            out.data_ptr(), ldy, ends_ptr, groups, rows, n, k, flags, kernel_id, _launch.stream_handle(device), status_ptr)
    if rc:
        _native.check(rc, "kmcts_mxfp4_gemm")
    return out


__all__ = ["BLOCK", "MXFP4Tensor", "mxfp4_dequantize", "mxfp4_gemm", "mxfp4_quantize"]
