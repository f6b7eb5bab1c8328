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
_CODES = (torch.uint8, torch.float4_e2m1fn_x2)
_SCALES = (torch.uint8, torch.float8_e8m0fnu)


class MXFP4Tensor(NamedTuple):
    """Packed codes and block scales; ``shape`` is the logical one."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], 2 * self.codes.shape[-1])


def _check_pair(name: str, q: MXFP4Tensor, dims: int, device: torch.device | None = None) -> None:
    _launch.check_tensor(f"{name} codes", q.codes, dims, _CODES, device)
    _launch.check_tensor(f"{name} scales", q.scales, dims, _SCALES, q.codes.device)
    k = 2 * q.codes.shape[-1]
    if k % BLOCK != 0:
        raise ValueError(f"{name} has K={k}, not a multiple of {BLOCK}")
    want = (*q.codes.shape[:-1], k // BLOCK)
    if tuple(q.scales.shape) != want:
        raise ValueError(f"{name} scales must have shape {want}, got {tuple(q.scales.shape)}")


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
    if x.dim() < 1 or x.shape[-1] % BLOCK != 0:
        raise ValueError(f"x must have a last dimension that is a multiple of {BLOCK}, got shape {tuple(x.shape)}")
    flat = _rows("x", x)
    _launch.check_tensor("x", flat, 2, tuple(_TYPES))
    device = x.device
    rows, k = flat.shape
    ldx = _launch.row_stride("x", flat, 0, BLOCK)
    caller = _launch.caller_stream(device, stream)
    with _launch.on_device(device, stream):
        if out is None:
            lead = x.shape[:-1]
            out = MXFP4Tensor(torch.empty((*lead, k // 2), dtype=torch.uint8, device=device),
                              torch.empty((*lead, k // BLOCK), dtype=torch.uint8, device=device))
            for t in out:
                _launch.share_result(t, caller)
        else:
            _check_pair("out", out, x.dim(), device)
            if out.shape != tuple(x.shape):
                raise ValueError(f"out must have shape {tuple(x.shape)}, got {out.shape}")
        codes, scales = _rows("out codes", out.codes), _rows("out scales", out.scales)
        rc = _native.load().kmcts_mxfp4_quantize(
            flat.data_ptr(), _TYPES[x.dtype], ldx, codes.data_ptr(), _launch.row_stride("out codes", codes, 0, 16),
            scales.data_ptr(), _launch.row_stride("out scales", scales, 0, 1), rows, k,
            _launch.stream_handle(device, stream))
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
    _check_pair("q", q, q.codes.dim())
    device = q.codes.device
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16
    if dtype not in _TYPES:
        raise TypeError(f"values must be bfloat16, float16 or float32, got {dtype}")
    codes, scales = _rows("codes", q.codes), _rows("scales", q.scales)
    rows, k = codes.shape[0], 2 * codes.shape[1]
    ldc, lds = _launch.row_stride("codes", codes, 0, 16), _launch.row_stride("scales", scales, 0, 1)
    caller = _launch.caller_stream(device, stream)
    with _launch.on_device(device, stream):
        if out is None:
            out = torch.empty(q.shape, dtype=dtype, device=device)
            _launch.share_result(out, caller)
        else:
            _launch.check_tensor("out", out, q.codes.dim(), (dtype,), device)
            if tuple(out.shape) != q.shape:
                raise ValueError(f"out must have shape {q.shape}, got {tuple(out.shape)}")
        flat = _rows("out", out)
        rc = _native.load().kmcts_mxfp4_dequantize(
            codes.data_ptr(), ldc, scales.data_ptr(), lds, flat.data_ptr(), _TYPES[dtype],
            _launch.row_stride("out", flat, 0, BLOCK), rows, k, _launch.stream_handle(device, stream))
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
    group's weight, as in :func:`kernel_mcts_b200.grouped.grouped_gemm`.
    """
    device = a.codes.device
    _check_pair("a", a, 2)
    _check_pair("b", b, 2 if ends is None else 3, device)
    rows, k = a.codes.shape[0], 2 * a.codes.shape[1]
    if 2 * b.codes.shape[-1] != k:
        raise ValueError(f"inner dimensions differ: a has K={k}, b has K={2 * b.codes.shape[-1]}")
    n = b.codes.shape[-2]
    groups, ends_ptr = 1, None
    if ends is not None:
        groups, ends_ptr = _launch.check_groups(ends, device), ends.data_ptr()
        if b.codes.shape[0] != groups:
            raise ValueError(f"b holds {b.codes.shape[0]} groups, ends {groups}")
    lda, ldas = _launch.row_stride("a codes", a.codes, 0, 16), _launch.row_stride("a scales", a.scales, 0, 1)
    ldb, ldbs = _launch.row_stride("b codes", b.codes, -2, 16), _launch.row_stride("b scales", b.scales, -2, 1)
    strides = (b.codes.stride(0), b.scales.stride(0)) if groups > 1 else (0, 0)
    status_ptr = _launch.status_pointer(status, device)
    kernel_id = kernel_code(kernel)
    caller = _launch.caller_stream(device, stream)
    with _launch.on_device(device, stream):
        flags = 0
        if out is None:
            out = torch.empty((rows, n), dtype=torch.bfloat16, device=device)
            _launch.share_result(out, caller)
            flags = _native.GROUPED_ZERO_REST
        else:
            _launch.check_tensor("out", out, 2, (torch.bfloat16,), device)
            if out.shape[0] != rows or out.shape[1] != n:
                raise ValueError(f"out must have shape {(rows, n)}, got {tuple(out.shape)}")
        rc = _native.load().kmcts_mxfp4_gemm(
            a.codes.data_ptr(), lda, a.scales.data_ptr(), ldas, b.codes.data_ptr(), strides[0], ldb,
            b.scales.data_ptr(), strides[1], ldbs, out.data_ptr(), _launch.row_stride("out", out, 0, 8), ends_ptr, groups,
            rows, n, k, flags, kernel_id, _launch.stream_handle(device, stream), status_ptr)
    _native.check(rc, "kmcts_mxfp4_gemm")
    return out


__all__ = ["BLOCK", "MXFP4Tensor", "mxfp4_dequantize", "mxfp4_gemm", "mxfp4_quantize"]
