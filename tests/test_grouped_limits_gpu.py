"""Expert-layer calls at the largest sizes that they accept."""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import grouped, mxfp4

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


# Contractions that one CTA works on for longer than the two seconds that a wait
# for a single stage may last.  Everything is zero but a few places, so sums are
# exact integers.


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kernel,k", [("pair", 2 ** 30), ("split", LARGEST)])  # 3.7 and 2.5 s
def test_product_over_a_long_row(cuda_device, kernel, k):
    x, w = (torch.zeros(1, k, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = torch.tensor([0, 77, k // 2 + 5, k - 1], device="cuda")
    x[0, at] = torch.tensor([1, 2, 3, 4], dtype=torch.bfloat16, device="cuda")
    w[0, at] = torch.tensor([5, -6, 7, 8], dtype=torch.bfloat16, device="cuda")
    status = status_word()
    y = grouped.grouped_gemm(x, w[None], torch.ones(1, dtype=torch.int32, device="cuda"), kernel=kernel, status=status)
    assert y.item() == 5 - 12 + 21 + 32 and status.item() == 0


def test_mxfp4_product_over_a_long_row(cuda_device):  # 3.1 s
    codes = torch.zeros(1, LARGEST // 2, dtype=torch.uint8, device="cuda")
    codes[0, torch.tensor([0, 77, LARGEST // 4 + 5, LARGEST // 2 - 1], device="cuda")] = 0x42  # 1 and 2
    a = mxfp4.MXFP4Tensor(codes, torch.full((1, LARGEST // 32), 127, dtype=torch.uint8, device="cuda"))
    status = status_word()
    y = mxfp4.mxfp4_gemm(a, a, kernel="pair", status=status)
    assert y.item() == 4 * (1 + 4) and status.item() == 0


def test_gradient_of_a_long_group(cuda_device):  # 2.5 s
    rows = 2 ** 29
    dy = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 77, rows // 2 + 5, rows - 18], device="cuda")
    dy[at] = torch.arange(32, device="cuda").view(4, 8).to(torch.bfloat16)
    dy[-17:] = float("nan")  # behind the group, in its last stage
    want = dy[at].double().T @ dy[at].double()
    status = status_word()
    dw = grouped.grouped_gemm_wgrad(dy, dy, torch.tensor([rows - 17], dtype=torch.int32, device="cuda"),
                                    dtype=torch.float32, kernel="tcgen05", status=status)
    assert torch.equal(dw[0].double(), want) and status.item() == 0
