"""grouped_linear and the calls beside it within torch's autograd: what is kept
for the backward pass, hooks, and results written into the caller's tensors."""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import grouped

pytestmark = pytest.mark.gpu


def operands(rows, n, k):
    """Small integers, two groups."""
    gen = torch.Generator().manual_seed(rows)
    x = torch.randint(-2, 3, (rows, k), generator=gen).to(torch.bfloat16).cuda()
    w = torch.randint(-2, 3, (2, n, k), generator=gen).to(torch.bfloat16).cuda()
    return x, w, torch.tensor([rows // 3, rows], dtype=torch.int32).cuda()


@pytest.mark.parametrize("frozen", ["w", "x"])
def test_only_what_the_backward_pass_reads_is_kept(cuda_device, frozen):
    """With a frozen weight the activations go as soon as their owner lets go
    of them, with frozen activations the weight does."""
    x, w, ends = operands(4096, 2048, 2048)  # x and w 16 MiB each
    x = (x.requires_grad_() if frozen == "w" else x) * 1  # not leaves, which torch itself keeps
    w = (w.requires_grad_() if frozen == "x" else w) * 1
    y = grouped.grouped_linear(x, w, ends)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    if frozen == "w":
        del x
    else:
        del w
    assert before - torch.cuda.memory_allocated() == 16 << 20
    y.sum().backward()
