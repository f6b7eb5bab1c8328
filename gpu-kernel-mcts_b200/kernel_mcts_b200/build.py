"""Builds the native parts of kernel_mcts_b200 in-tree with nvcc (sm_100a).

Outputs (git-ignored, shipped with the source tree):
  _lib/libkmcts_gemm_sm100.so   the C-ABI library (include/kmcts_gemm.h, kmcts_grouped.h)
  _lib/kmcts_bf16_eval          the evaluation harness executable built on it
  _lib/kmcts_torch_calls.so     the expert-layer calls on torch tensors (host code)

Run as ``python -m kernel_mcts_b200.build`` (with gpu-kernel-mcts_b200/ on
sys.path) or call :func:`build_all`.  Rebuilds only what is older than its
sources.
"""

from __future__ import annotations

import concurrent.futures
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
REPO_ROOT = PACKAGE_DIR.parent.parent
CSRC = PACKAGE_DIR / "csrc"
LIB_DIR = PACKAGE_DIR / "_lib"
INCLUDE = REPO_ROOT / "include"
OBJ_DIR = LIB_DIR / "obj"

LIBRARY = LIB_DIR / "libkmcts_gemm_sm100.so"
HARNESS = LIB_DIR / "kmcts_bf16_eval"
TORCH_CALLS = LIB_DIR / "kmcts_torch_calls.so"
TORCH_CALLS_BUILT_FOR = LIB_DIR / "kmcts_torch_calls.built_for"  # torch_and_python() at the time

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON_FLAGS = ["-std=c++17", "-O3", "-lineinfo", *ARCH_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}"]

LIBRARY_SOURCES = ("gemm_tcgen05.cu", "gemm_tcgen05_pair.cu", "gemm_tcgen05_stream.cu", "gemm_simt.cu", "compare.cu",
                   "capi.cu", "ipc.cu", "selftest.cu", "workspace.cu", "host_gemm.cu")
GROUPED_SOURCES = ("grouped_api.cu", "grouped_pair.cu", "grouped_split.cu", "grouped_simt.cu", "mxfp4_quantize.cu")
HEADERS = ("ptx_sm100.cuh", "gemm_common.cuh", "kmcts_internal.h")
GROUPED_HEADERS = ("grid_walk.h", "grouped_common.cuh", "grouped_internal.h", "grouped_tiles.cuh", "ptx_grouped.cuh")


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the sm_100a build needs the CUDA toolkit")
    return found


def _newest(paths) -> float:
    return max(Path(p).stat().st_mtime for p in paths)


def _stale(target: Path, deps) -> bool:
    return not target.exists() or target.stat().st_mtime < _newest(deps)


def _run(command: list[str]) -> None:
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(
            "build step failed:\n" + " ".join(command) + "\n" + result.stdout + result.stderr
        )


def build_library(verbose: bool = False) -> Path:
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    headers = [CSRC / h for h in HEADERS] + [INCLUDE / "kmcts_gemm.h"]
    jobs = []
    objects = []
    grouped_headers = [*headers, *(CSRC / h for h in GROUPED_HEADERS), INCLUDE / "kmcts_grouped.h"]
    for name in (*LIBRARY_SOURCES, *GROUPED_SOURCES):
        src = CSRC / name
        obj = OBJ_DIR / (Path(name).stem + ".o")
        objects.append(obj)
        if _stale(obj, [src, *(grouped_headers if name in GROUPED_SOURCES else headers), Path(__file__)]):
            jobs.append([nvcc(), *COMMON_FLAGS, "-Xcompiler", "-fPIC", "-c", str(src), "-o", str(obj)])
    if jobs:
        with concurrent.futures.ThreadPoolExecutor(max_workers=len(jobs)) as pool:
            for cmd, fut in [(cmd, pool.submit(_run, cmd)) for cmd in jobs]:
                if verbose:
                    print(" ".join(cmd), file=sys.stderr)
                fut.result()
    if _stale(LIBRARY, objects):
        _run([nvcc(), *ARCH_FLAGS, "-shared", "-o", str(LIBRARY), *map(str, objects)])
    return LIBRARY


def cutlass_include() -> Path | None:
    """CUTLASS headers vendored in this image (flashinfer's copy), if present.
    Used only for the CUTLASS column of the vendor baselines."""
    import importlib.util

    spec = importlib.util.find_spec("flashinfer")
    if spec is None or spec.origin is None:
        return None
    path = Path(spec.origin).parent / "data" / "cutlass" / "include"
    return path if (path / "cutlass" / "gemm" / "device" / "gemm.h").exists() else None


def build_harness(verbose: bool = False) -> Path:
    src = CSRC / "harness.cu"
    if not src.exists():
        return HARNESS
    lib = build_library(verbose)
    sources = [src]
    flags = ["-DKMCTS_HAVE_CUTLASS=0"]
    cutlass = cutlass_include()
    if cutlass is not None:
        sources.append(CSRC / "vendor_cutlass.cu")
        flags = ["-DKMCTS_HAVE_CUTLASS=1", f"-I{cutlass}"]
    if _stale(HARNESS, [*sources, lib, INCLUDE / "kmcts_gemm.h", Path(__file__)]):
        cmd = [
            nvcc(), *COMMON_FLAGS, *flags, *map(str, sources), "-o", str(HARNESS),
            f"-L{LIB_DIR}", "-lkmcts_gemm_sm100", "-lcublas",
            "-Xlinker", f"-rpath={LIB_DIR}", "-Xlinker", "-rpath=$ORIGIN",
        ]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        _run(cmd)
    return HARNESS


def torch_dir() -> Path | None:
    """The installed torch, if it has C++ headers and was built with CUDA."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        return None
    found = Path(spec.origin).parent
    needed = ("include/c10/cuda/CUDAStream.h", "include/torch/csrc/utils/pybind.h", "lib/libc10_cuda.so")
    return found if all((found / name).exists() for name in needed) else None


def torch_and_python() -> str:
    """What a module built against torch's C++ headers depends on."""
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a tree on the path, not an installed package
        import torch

        version = torch.__version__
    return f"torch {version}, {sys.implementation.cache_tag}"


def torch_calls_built_for() -> str | None:
    return TORCH_CALLS_BUILT_FOR.read_text() if TORCH_CALLS_BUILT_FOR.exists() else None


def build_torch_calls(verbose: bool = False) -> Path:
    """The torch-facing calls: host code only, against this interpreter's torch."""
    lib = build_library(verbose)
    src = CSRC / "torch_calls.cpp"
    headers = (INCLUDE / "kmcts_grouped.h", INCLUDE / "kmcts_gemm.h")
    torch = torch_dir()
    if torch is None:
        raise RuntimeError("no torch with CUDA and C++ headers; the expert-layer calls are built against them")
    target = torch_and_python()
    if torch_calls_built_for() == target and not _stale(TORCH_CALLS, [src, *headers, Path(__file__)]):
        return TORCH_CALLS
    includes = [torch / "include", torch / "include" / "torch" / "csrc" / "api" / "include",
                Path(sysconfig.get_paths()["include"]), Path(nvcc()).resolve().parent.parent / "include"]
    cmd = [
        shutil.which("g++") or "g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", f"-I{INCLUDE}",
        *(arg for path in includes for arg in ("-isystem", str(path))), str(src), "-o", str(TORCH_CALLS),
        f"-L{LIB_DIR}", f"-l{lib.stem.removeprefix('lib')}", f"-L{torch / 'lib'}",
        *(f"-l{name}" for name in ("c10", "c10_cuda", "torch", "torch_cpu", "torch_cuda", "torch_python")),
        "-Wl,-rpath,$ORIGIN",
    ]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    TORCH_CALLS_BUILT_FOR.unlink(missing_ok=True)
    _run(cmd)
    TORCH_CALLS_BUILT_FOR.write_text(target)
    return TORCH_CALLS


def build_all(verbose: bool = False) -> None:
    """Everything that can be built here: the library and the harness need nvcc
    alone, the torch calls a torch with CUDA and its headers too."""
    build_library(verbose)
    build_harness(verbose)
    if torch_dir() is not None:
        build_torch_calls(verbose)
    else:
        print("no torch with CUDA and C++ headers: the expert-layer calls on torch tensors are not built", file=sys.stderr)


if __name__ == "__main__":
    build_all(verbose=True)
    print(LIBRARY)
