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

:func:`grouped_gemm` and :func:`grouped_gemm_wgrad` are not recorded by
autograd: their results require no gradient, whatever the operands do, and an
``out`` that requires one is refused while autograd records.  A write into
``out`` counts as an in-place change.
"""

from __future__ import annotations

import torch

from . import _launch, _native
from .gemm import layout_code

KERNELS = {"auto": _native.KERNEL_AUTO, "tcgen05": _native.KERNEL_TCGEN05, "simt": _native.KERNEL_SIMT,
           "pair": _native.KERNEL_GROUPED_PAIR, "split": _native.KERNEL_GROUPED_SPLIT}
_GRADIENT_KERNELS = {name: KERNELS[name] for name in ("auto", "tcgen05", "simt")}

_calls = _native.torch_calls


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
    args = (x, w, ends, out, layout_code(w_layout), kernel_code(kernel), status)
    if stream is None:
        return _calls.grouped_gemm(*args)
    return _launch.run_on(stream, (x, w, ends, out, status), _calls.grouped_gemm, *args)


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
    several micro-batches; an empty group then leaves its part as it was, and
    is zeros otherwise.
    """
    args = (dy, x, ends, out, dtype, accumulate, kernel_code(kernel, _GRADIENT_KERNELS), status)
    if stream is None:
        return _calls.grouped_gemm_wgrad(*args)
    return _launch.run_on(stream, (dy, x, ends, out, status), _calls.grouped_gemm_wgrad, *args)


def grouped_linear(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, *, w_layout: str | int = "col") -> torch.Tensor:
    """Differentiable ``grouped_gemm(x, w, ends, w_layout=w_layout)``.

    The gradients of ``x`` and ``w`` are bfloat16; ``x``'s is zero in rows
    behind the last group.  Of ``x`` and ``w`` only what the wanted gradients
    read is kept.  Once differentiable: a backward pass with ``create_graph=True``
    is refused.  As with any torch function, a
    backward pass may be captured into a CUDA graph only while no autograd
    graph of the same leaves from outside the capture is alive."""
    return _calls.grouped_linear(x, w, ends, layout_code(w_layout))


__all__ = ["grouped_gemm", "grouped_gemm_wgrad", "grouped_linear"]
