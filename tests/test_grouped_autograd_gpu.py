"""grouped_linear and the calls beside it within torch's autograd: what is kept
for the backward pass, hooks, and results written into the caller's tensors."""

from __future__ import annotations

import contextlib
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from kernel_mcts_b200 import grouped, mxfp4

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


def writers():
    """Each call that writes into the caller's tensors: those, and the call."""
    x, w, ends = operands(64, 32, 64)
    q = mxfp4.mxfp4_quantize(x)
    y, dw = torch.zeros(64, 32, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 32, 64, device="cuda")
    back = torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
    into = mxfp4.MXFP4Tensor(torch.zeros_like(q.codes), torch.zeros_like(q.scales))
    return {
        "grouped_gemm": ([y], lambda: grouped.grouped_gemm(x, w, ends, y)),
        "grouped_gemm_wgrad": ([dw], lambda: grouped.grouped_gemm_wgrad(x[:, :32], x, ends, dw, accumulate=True)),
        "mxfp4_quantize": (into, lambda: mxfp4.mxfp4_quantize(x, into)),
        "mxfp4_dequantize": ([back], lambda: mxfp4.mxfp4_dequantize(q, back)),
        "mxfp4_gemm": ([y], lambda: mxfp4.mxfp4_gemm(q, mxfp4.mxfp4_quantize(w[0]), out=y)),
    }


@pytest.mark.parametrize("name", ["grouped_gemm", "grouped_gemm_wgrad", "mxfp4_quantize", "mxfp4_dequantize", "mxfp4_gemm"])
def test_a_write_into_the_callers_tensor_counts_as_one(cuda_device, name):
    tensors, call = writers()[name]
    before = [t._version for t in tensors]
    call()
    assert all(t._version > v for t, v in zip(tensors, before))
    with torch.inference_mode():
        tensors, call = writers()[name]  # inference tensors, which count no versions
        call()


def test_a_saved_tensor_that_a_call_overwrites_is_noticed(cuda_device):
    x, w, ends = operands(64, 32, 64)
    y = torch.ones(64, 32, dtype=torch.bfloat16, device="cuda")
    scale = torch.ones(64, 32, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    loss = (scale * y).sum()  # keeps y
    grouped.grouped_gemm(x, w, ends, y[:, :32])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    kept = grouped.grouped_linear(x.requires_grad_() * 1, w.requires_grad_() * 1, ends)
    ends.copy_(ends)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


@pytest.mark.parametrize("name", ["grouped_gemm", "grouped_gemm_wgrad", "mxfp4_dequantize", "mxfp4_gemm"])
def test_results_that_require_a_gradient_are_not_written(cuda_device, name):
    """Into a value that the autograd graph computed, or a leaf of it."""
    tensors, call = writers()[name]
    tensors[0].requires_grad_()
    with pytest.raises(ValueError, match="must not require a gradient"):
        call()
    assert (tensors[0] == 0).all()
    with torch.no_grad():
        call()
    assert not (tensors[0] == 0).all()


def gradients(x, w, ends, dy, around):
    """(y, dx, dw) of a step within a context, from leaves of its own."""
    x, w = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    with around:
        y = grouped.grouped_linear(x, w, ends)
    y.backward(dy)
    return y.detach(), x.grad, w.grad


def test_saved_tensor_hooks_and_checkpointing(cuda_device):
    """What is kept may be moved to the host and back, or computed again."""
    x, w, ends = operands(200, 136, 72)
    dy = operands(200, 136, 136)[0]
    plain = gradients(x, w, ends, dy, contextlib.nullcontext())
    moved = gradients(x, w, ends, dy, torch.autograd.graph.save_on_cpu())
    assert all(torch.equal(a, b) for a, b in zip(plain, moved))
    for reentrant in (False, True):
        x2, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = checkpoint(lambda a, b: grouped.grouped_linear(a, b, ends), x2, w2, use_reentrant=reentrant)
        y.backward(dy)
        assert all(torch.equal(a, b) for a, b in zip(plain, (y.detach(), x2.grad, w2.grad)))


def test_steps_on_two_threads_and_streams(cuda_device):
    x, w, ends = operands(200, 136, 72)
    dy = operands(200, 136, 136)[0]
    plain = gradients(x, w, ends, dy, contextlib.nullcontext())
    torch.cuda.synchronize()

    def steps(_):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results = [gradients(x, w, ends, dy, contextlib.nullcontext()) for _ in range(20)]
        stream.synchronize()
        return all(torch.equal(a, b) for result in results for a, b in zip(plain, result))

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(steps, range(4)))


def test_gradients_of_one_weight_shared_by_all_groups(cuda_device):
    """An expanded weight's gradient is the sum over the groups."""
    x, w, ends = operands(200, 136, 72)
    dy = operands(200, 136, 136)[0]
    one = w[:1].clone().requires_grad_()
    y = grouped.grouped_linear(x, one.expand(2, 136, 72), ends)
    (got,) = torch.autograd.grad(y, one, dy)
    cut = int(ends[0])
    parts = [(dy[lo:hi].double().T @ x[lo:hi].double()).to(torch.bfloat16) for lo, hi in ((0, cut), (cut, 200))]
    assert torch.equal(got[0], parts[0] + parts[1])
