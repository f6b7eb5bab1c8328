"""Expert-layer calls that follow one another without waiting, each reading
what the one before wrote into buffers that all of them share."""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import mxfp4
from kernel_mcts_b200.mxfp4 import MXFP4Tensor

pytestmark = pytest.mark.gpu


def inputs(count, rows, k, dtype):
    """Small integers times a power of two of each block's own, a different one
    in every input: scales of one call serve no other."""
    gen = torch.Generator().manual_seed(rows + k)
    values = torch.randint(-6, 7, (count, rows, k), generator=gen).float()
    values[..., ::32] = 6  # every block reaches the largest code, so its values are exact
    values = torch.where(values.abs() == 5, 4.0, values)
    powers = torch.randint(-8, 9, (count, rows, k // 32), generator=gen)
    return torch.ldexp(values, powers.repeat_interleave(32, -1)).to(dtype).cuda()


def buffers(rows, k):
    return MXFP4Tensor(torch.zeros(rows, k // 2, dtype=torch.uint8, device="cuda"),
                       torch.zeros(rows, k // 32, dtype=torch.uint8, device="cuda"))


def directly_and_as_a_graph(run, results, wanted):
    run()
    torch.cuda.synchronize()
    for got, want in zip(results, wanted):
        assert torch.equal(got, want)
    for got in results:
        got.fill_(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(results, wanted):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k", [(3, 96), (70, 4096), (1000, 2048)])
def test_quantise_and_restore_through_one_buffer(cuda_device, dtype, rows, k):
    xs, q = inputs(12, rows, k, dtype), buffers(rows, k)
    results = [torch.zeros(rows, k, dtype=dtype, device="cuda") for _ in xs]

    def run():
        for x, result in zip(xs, results):
            mxfp4.mxfp4_quantize(x, q)
            mxfp4.mxfp4_dequantize(q, result)

    directly_and_as_a_graph(run, results, xs)


@pytest.mark.parametrize("kernel", ["pair", "split", "simt"])
@pytest.mark.parametrize("rows,k,odd", [(3, 96, 0), (70, 4096, 3), (400, 1024, 0)])
def test_quantise_and_multiply_through_one_buffer(cuda_device, kernel, rows, k, odd):
    """The weight picks one element of each row, so an output is one input and
    a scale of another call shows.  odd: scales that start at an odd address."""
    n = 136
    xs, q = inputs(12, rows, k, torch.bfloat16), buffers(rows, k)
    if odd:
        q = q._replace(scales=torch.zeros(rows, k // 32 + 8, dtype=torch.uint8, device="cuda")[:, odd:odd + k // 32])
    at = torch.arange(n) * 37 % k
    w = torch.zeros(n, k)
    w[torch.arange(n), at] = 1
    w = mxfp4.mxfp4_quantize(w.cuda())
    results = [torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda") for _ in xs]

    def run():
        for x, result in zip(xs, results):
            mxfp4.mxfp4_quantize(x, q)
            mxfp4.mxfp4_gemm(q, w, out=result, kernel=kernel)

    directly_and_as_a_graph(run, results, [x[:, at.cuda()] for x in xs])
