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


@pytest.mark.parametrize("kernel", ["tcgen05", "simt"])
@pytest.mark.parametrize("dtype,accumulate", [(torch.bfloat16, False), (torch.float32, False), (torch.float32, True)])
def test_groups_side_by_side_in_every_row(cuda_device, kernel, dtype, accumulate):
    """A main gradient kept as [N, groups, K]: its groups interleave but share nothing."""
    counts, n, k = [70, 0, 130], 136, 72
    gen = torch.Generator().manual_seed(1)
    dy, x = (torch.randint(-2, 3, (200, c), generator=gen).to(torch.bfloat16).cuda() for c in (n, k))
    ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    store = torch.full((n, 4, k), 3, dtype=dtype, device="cuda")
    out = store[:, :3].transpose(0, 1)
    assert out.shape == (3, n, k) and out.stride(0) == k
    grouped.grouped_gemm_wgrad(dy, x, ends, out, accumulate=accumulate, kernel=kernel)
    want = torch.stack([dy[:70].double().T @ x[:70].double(), torch.zeros(n, k, device="cuda").double(),
                        dy[70:].double().T @ x[70:].double()])
    assert torch.equal(out, (want + (3 if accumulate else 0)).to(dtype))
    assert (store[:, 3] == 3).all()


def test_groups_that_overlap_are_refused(cuda_device):
    dy, x = torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")
    ends = torch.tensor([2, 4], dtype=torch.int32, device="cuda")
    store = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    for strides in ((0, 16, 1), (8, 32, 1), (16, 24, 1), (7 * 16, 16, 1)):
        with pytest.raises(ValueError, match="overlapping groups"):
            grouped.grouped_gemm_wgrad(dy, x, ends, store.as_strided((2, 8, 16), strides))
    for strides in ((16, 32, 1), (128, 16, 1), (7 * 32 + 16, 32, 1)):
        grouped.grouped_gemm_wgrad(dy, x, ends, store.as_strided((2, 8, 16), strides))
