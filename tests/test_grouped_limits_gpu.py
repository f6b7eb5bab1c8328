"""Expert-layer calls at the largest sizes that they accept."""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import grouped

pytestmark = pytest.mark.gpu

LARGEST = 2 ** 31 - 1024


@pytest.mark.parametrize("behind", [0, 3, 5000])
def test_as_many_rows_as_there_may_be(cuda_device, behind):
    """One column each way: the CUDA-core kernel, whose grid's step passes 2^31
    from the last rows.  Doubling is exact in BF16."""
    x = torch.arange(LARGEST, dtype=torch.int32, device="cuda").bitwise_and_(127).to(torch.bfloat16)[:, None]
    w = torch.full((1, 1, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    ends = torch.tensor([LARGEST - behind], dtype=torch.int32, device="cuda")
    y = grouped.grouped_gemm(x, w, ends)
    x.mul_(2)
    if behind:
        x[-behind:] = 0
    assert torch.equal(y, x)
