"""Index arithmetic of the expert-layer kernels at the largest sizes that their
entry points accept, compiled for the host."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "gpu-kernel-mcts_b200" / "kernel_mcts_b200" / "csrc"
LARGEST = 2 ** 31 - 1024

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "grid_walk.h"
int main(int argc, char** argv) {
    const long long first = atoll(argv[1]), end = atoll(argv[2]);
    const unsigned blocks = static_cast<unsigned>(atoll(argv[3]));
    for (unsigned b = 0; b < blocks; ++b) {
        long long count = 0, low = end, high = -1;
        for (kmcts::grouped::GridWalk w(first, end, b, blocks); w.more() && count < 1000000; w.next()) {
            ++count;
            if (w.at < low) low = w.at;
            if (w.at > high) high = w.at;
        }
        std::printf("%lld %lld %lld\n", count, low, high);
    }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    compiler = shutil.which("g++") or shutil.which("c++")
    assert compiler, "the native build needs a C++ compiler"
    at = tmp_path_factory.mktemp("walk")
    (at / "walk.cpp").write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{CSRC}", str(at / "walk.cpp"), "-o", str(at / "walk")], check=True, timeout=300)

    def run(first, end, blocks):
        out = subprocess.run([str(at / "walk"), *map(str, (first, end, blocks))], check=True, capture_output=True,
                             text=True, timeout=60).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


@pytest.mark.parametrize("first,end", [(0, 0), (0, 5), (LARGEST, LARGEST), (LARGEST - 1, LARGEST),
                                       (LARGEST - 5000, LARGEST), (2 ** 31 - 3000, 2 ** 31 - 1)])
@pytest.mark.parametrize("blocks", [1, 148, 1184])
def test_blocks_share_out_all_the_work_and_no_more(walk, first, end, blocks):
    """1184: eight blocks on each of 148 SMs.  In 32 bits a block's first item
    can pass 2^31, and is below the end again."""
    for b, (count, low, high) in enumerate(walk(first, end, blocks)):
        items = range(first + b, end, blocks)
        assert count == len(items)
        assert not items or (low, high) == (items[0], items[-1])
