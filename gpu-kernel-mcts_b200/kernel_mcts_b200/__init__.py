"""kernel_mcts_b200: the B200-native (sm_100a) BF16 GEMM hot path of kernel_mcts,
and the matrix products of expert layers.

The GEMM, its correctness check and its timing protocol run in hand-written
CUDA (libkmcts_gemm_sm100.so, C ABI in include/kmcts_gemm.h); Python only
allocates device memory and wires the reference's evaluation contract on top.
:mod:`kernel_mcts_b200.grouped` has the BF16 products grouped by expert with
their gradients, :mod:`kernel_mcts_b200.mxfp4` microscaled 4-bit quantisation
and products (include/kmcts_grouped.h), both on torch tensors.
"""

from ._native import (
    B_COL,
    B_ROW,
    GemmConfig,
    KmctsError,
    NativeLibraryError,
    config_legal,
    config_smem_bytes,
    default_config,
    launch_count,
    make_config,
    select_config,
    version,
)

__all__ = [
    "B_COL",
    "B_ROW",
    "GemmConfig",
    "KmctsError",
    "NativeLibraryError",
    "config_legal",
    "config_smem_bytes",
    "default_config",
    "launch_count",
    "make_config",
    "select_config",
    "version",
]
