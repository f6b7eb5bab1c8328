"""BF16 products grouped by expert, and their gradients.

Rows are sorted by group: ``ends`` is an int32 tensor on the operands' device
whose element ``e`` is one past the last row of group ``e`` (the row counts'
running sum).  It is read on the device; no call waits for it.  Ends that
decrease or exceed the rows only make groups empty or short.  Rows behind the
last end belong to no group: results that the call allocates hold zeros there,
an ``out`` that the caller gives is left as it was.

The weight of group ``e`` is ``w[e]``: ``[N, K]`` for ``w_layout="col"``
(``Y = X·W^T``, the column-major B of the dense GEMM) or ``[K, N]`` for
``"row"`` (``Y = X·W``).  ``grouped_gemm(dy, w, ends, w_layout="row")`` on the
weight of a ``"col"`` product is that product's input gradient,
:func:`grouped_gemm_wgrad` its weights' gradient, and :func:`grouped_linear`
ties the three together for autograd.
"""

from __future__ import annotations

import torch

from . import _launch, _native
from .gemm import layout_code

KERNELS = {"auto": _native.KERNEL_AUTO, "tcgen05": _native.KERNEL_TCGEN05, "simt": _native.KERNEL_SIMT,
           "pair": _native.KERNEL_GROUPED_PAIR, "split": _native.KERNEL_GROUPED_SPLIT}
_GRADIENT_KERNELS = {name: KERNELS[name] for name in ("auto", "tcgen05", "simt")}

_BF16 = (torch.bfloat16,)
_GRADIENT_TYPES = {torch.bfloat16: _native.TYPE_BF16, torch.float32: _native.TYPE_FP32}


def kernel_code(kernel: str, kernels: dict[str, int] = KERNELS) -> int:
    try:
        return kernels[kernel]
    except KeyError as error:
        raise ValueError(f"unknown kernel {kernel!r}; use one of {sorted(kernels)}") from error


def grouped_gemm(
    x: torch.Tensor,
    w: torch.Tensor,
    ends: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    w_layout: str | int = "col",
    kernel: str = "auto",
    stream: torch.cuda.Stream | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """Each row of ``x`` ``[rows, K]`` times its group's weight: ``[rows, N]``.

    Rows may be strided; FP32 sums, one rounding.  ``kernel`` is ``"auto"``,
    ``"tcgen05"`` (``"pair"`` or ``"split"`` by size: CTA pairs, or clusters that
    split K for few rows; 16-byte aligned rows) or ``"simt"`` (any operands).
    Asynchronous on ``stream``
    (the current one by default).  ``status`` is as for
    :func:`kernel_mcts_b200.gemm.bf16_gemm`.
    """
    code = layout_code(w_layout)
    device = x.get_device()
    (rows, k), _, ldx = _launch.rows_of("x", x, 2, _BF16, device, 8)
    w_shape, w_strides, ldw = _launch.rows_of("w", w, 3, _BF16, device, 8)
    groups = _launch.check_groups(ends, device)
    n, kw = (w_shape[1], w_shape[2]) if code == _native.B_COL else (w_shape[2], w_shape[1])
    if kw != k:
        raise ValueError(f"inner dimensions differ: x has K={k}, w has K={kw}")
    if w_shape[0] != groups:
        raise ValueError(f"w holds {w_shape[0]} groups, ends {groups}")
    _launch.check_sizes(rows, n, k)
    status_ptr = _launch.status_pointer(status, device)
    kernel_id = kernel_code(kernel)
    caller = _launch.caller_stream(device, stream)
    _launch.use_on(stream, caller, x, w, ends, out, status)
    with _launch.on_device(device, stream):
        if out is None:
            out = _launch.share_result(x.new_empty((rows, n)), caller)
            ldy, flags = n, _native.GROUPED_ZERO_REST
        else:
            shape, _, ldy = _launch.rows_of("out", out, 2, _BF16, device, 8)
            if shape != (rows, n):
                raise ValueError(f"out must have shape {(rows, n)}, got {tuple(shape)}")
            flags = 0
        rc = _native.load().kmcts_bf16_grouped_gemm(
            x.data_ptr(), ldx, w.data_ptr(), w_strides[0] if groups > 1 else 0, ldw, code, out.data_ptr(), ldy,
            ends.data_ptr(), groups, rows, n, k, flags, kernel_id, _launch.stream_handle(device), status_ptr)
    if rc:
        _native.check(rc, "kmcts_bf16_grouped_gemm")
    return out


def grouped_gemm_wgrad(
    dy: torch.Tensor,
    x: torch.Tensor,
    ends: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    dtype: torch.dtype | None = None,
    accumulate: bool = False,
    kernel: str = "auto",
    stream: torch.cuda.Stream | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """``dy[rows of e]^T · x[rows of e]`` for every group: ``[groups, N, K]``.

    The result is ``dtype`` (bfloat16 by default, or float32) or ``out``'s type.
    ``accumulate`` adds to a float32 ``out``, as for a main gradient kept over
    several micro-batches (sums below ``2^-126`` become zero); an empty group
    then leaves its part as it was, and is zeros otherwise.
    """
    device = dy.get_device()
    (rows, n), _, lddy = _launch.rows_of("dy", dy, 2, _BF16, device, 8)
    (x_rows, k), _, ldx = _launch.rows_of("x", x, 2, _BF16, device, 8)
    groups = _launch.check_groups(ends, device)
    if x_rows != rows:
        raise ValueError(f"dy has {rows} rows, x {x_rows}")
    _launch.check_sizes(rows, n, k)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16
    if dtype not in _GRADIENT_TYPES:
        raise TypeError(f"the gradient must be bfloat16 or float32, got {dtype}")
    if accumulate and (out is None or dtype != torch.float32):
        raise ValueError("accumulate needs a float32 out")
    status_ptr = _launch.status_pointer(status, device)
    kernel_id = kernel_code(kernel, _GRADIENT_KERNELS)
    caller = _launch.caller_stream(device, stream)
    _launch.use_on(stream, caller, dy, x, ends, out, status)
    with _launch.on_device(device, stream):
        if out is None:
            out = _launch.share_result(x.new_empty((groups, n, k), dtype=dtype), caller)
            ldo, group_stride = k, n * k
        else:
            shape, strides, ldo = _launch.rows_of("out", out, 3, (dtype,), device, 8)
            if shape != (groups, n, k):
                raise ValueError(f"out must have shape {(groups, n, k)}, got {tuple(shape)}")
            group_stride = strides[0] if groups > 1 else n * ldo
            if groups > 1 and n > 0 and group_stride < (n - 1) * ldo + k:
                raise ValueError("out has overlapping groups")
        rc = _native.load().kmcts_bf16_grouped_wgrad(
            dy.data_ptr(), lddy, x.data_ptr(), ldx, out.data_ptr(), group_stride, ldo, _GRADIENT_TYPES[dtype],
            int(accumulate), ends.data_ptr(), groups, rows, n, k, kernel_id, _launch.stream_handle(device), status_ptr)
    if rc:
        _native.check(rc, "kmcts_bf16_grouped_wgrad")
    return out


def _strided_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where the kernels can read it, else a contiguous copy (an
    expanded gradient, as a sum's backward gives, has overlapping rows)."""
    if t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, ends, code):
        ctx.save_for_backward(x, w, ends)
        ctx.code = code
        return grouped_gemm(x, w, ends, w_layout=code)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # create_graph: the gradients below would not be part of it
            raise RuntimeError("grouped_linear is differentiable once")
        x, w, ends = ctx.saved_tensors
        dy = _strided_rows(dy)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = grouped_gemm(dy, w, ends, w_layout=1 - ctx.code)
        if ctx.needs_input_grad[1]:
            dw = grouped_gemm_wgrad(dy, x, ends) if ctx.code == _native.B_COL else grouped_gemm_wgrad(x, dy, ends)
        return dx, dw, None, None


def grouped_linear(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, *, w_layout: str | int = "col") -> torch.Tensor:
    """Differentiable ``grouped_gemm(x, w, ends, w_layout=w_layout)``.

    The gradients of ``x`` and ``w`` are bfloat16; ``x``'s is zero in rows
    behind the last group.  Once differentiable.  As with any torch function, a
    backward pass may be captured into a CUDA graph only while no autograd
    graph of the same leaves from outside the capture is alive."""
    return _GroupedLinear.apply(x, w, ends, layout_code(w_layout))


__all__ = ["grouped_gemm", "grouped_gemm_wgrad", "grouped_linear"]
