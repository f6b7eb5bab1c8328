"""Weights' gradients added to an FP32 main gradient, bit by bit."""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import grouped

pytestmark = pytest.mark.gpu

# Main gradients at the ends of FP32's range and around its smallest normal number.
MAIN = [0.0, -0.0, 2.0 ** -149, -2.0 ** -149, 2.0 ** -127, -2.0 ** -127, 3 * 2.0 ** -128, 2.0 ** -126, -2.0 ** -126,
        1.5 * 2.0 ** -126, -1.5 * 2.0 ** -126, 2.0 ** -125, 1.0, -1.0, float("inf"), float("nan")]
# One row's output gradient; with an input of 2^-63 the sums reach from 2^-149 up.
ROW = [0.0, 2.0 ** -63, -2.0 ** -63, 2.0 ** -62, -2.0 ** -62, 2.0 ** -64, -2.0 ** -64, 2.0 ** -67, 2.0 ** -80, 2.0 ** -86,
       -2.0 ** -86, 1.0, 3.0, -3.0, float("inf"), float("nan")]


def same_bits(a, b):
    """NaN equals NaN, -0.0 does not equal 0.0."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num().view(torch.int32),
                                                             b.nan_to_num().view(torch.int32))


@pytest.mark.parametrize("kernel", ["tcgen05", "simt"])
def test_accumulate_rounds_once_and_leaves_empty_groups(cuda_device, kernel):
    dy = torch.tensor([ROW], device="cuda").to(torch.bfloat16)
    x = torch.full((1, 16), 2.0 ** -63, dtype=torch.bfloat16, device="cuda")
    main = torch.tensor(MAIN, device="cuda").expand(3, 16, 16).contiguous()
    before = main.clone()
    grouped.grouped_gemm_wgrad(dy, x, torch.tensor([0, 1, 1], dtype=torch.int32, device="cuda"), main, accumulate=True,
                               kernel=kernel)
    # Doubles hold each product and sum of one product exactly but for tiny
    # addends, where the FP32 rounding below is the only one that shows.
    want = (before[1].cpu().double() + dy.cpu().double().T @ x.cpu().double()).float()
    got = main.cpu()
    assert same_bits(got[1], want)
    assert torch.equal(got[0].view(torch.int32), before[0].cpu().view(torch.int32))
    assert torch.equal(got[2].view(torch.int32), before[2].cpu().view(torch.int32))


@pytest.mark.parametrize("kernel", ["tcgen05", "simt"])
def test_accumulate_over_no_rows_changes_nothing(cuda_device, kernel):
    main = torch.tensor(MAIN, device="cuda").expand(2, 16, 16).contiguous()
    before = main.clone()
    none = torch.zeros(0, 16, dtype=torch.bfloat16, device="cuda")
    grouped.grouped_gemm_wgrad(none, none, torch.zeros(2, dtype=torch.int32, device="cuda"), main, accumulate=True,
                               kernel=kernel)
    assert torch.equal(main.view(torch.int32), before.view(torch.int32))
