"""Products whose CTAs walk several tiles of several stages each: both
accumulators in turn, the ring of stages carried into the next tile, scales
fetched ahead for it, ragged last stages that meet the same barriers again.

Integer-valued operands: every FP32 sum is exact whatever its order, so outputs
are compared bit for bit with the 64-bit product, rounded once.
"""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import _native, grouped, mxfp4
from kernel_mcts_b200.mxfp4 import MXFP4Tensor

pytestmark = pytest.mark.gpu

# Row counts by group: empty, single rows, and both sides of 16, 64, 128, 192 and 256.
COUNTS = [0, 300, 17, 700, 256, 1, 513, 255, 64, 0, 1000, 33, 384, 129, 511, 90, 257, 640, 5, 193]
BEHIND = 11  # rows behind the last group


def ends_of(counts):
    return torch.tensor(counts).cumsum(0).to(torch.int32).cuda()


def integers(*shape, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=gen).to(torch.bfloat16).cuda()


def by_group(counts, rows, cols, times):
    """times(e, first row, row past the last) for each group, zeros behind."""
    out, lo = torch.zeros(rows, cols, dtype=torch.float64, device="cuda"), 0
    for e, c in enumerate(counts):
        out[lo:lo + c] = times(e, lo, lo + c)
        lo += c
    return out


def status_of(call, *args, **kwargs):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = call(*args, status=status, **kwargs)
    assert status.item() == 0
    return out


def check_walk(tiles, workers, times=3):
    """The case is as long as it says: that many tiles for each worker."""
    assert tiles >= times * workers


def multiprocessors():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("n,k", [(2568, 1000), (2560, 136), (2600, 64)])
def test_pairs_walk_many_tiles(cuda_device, layout, n, k):
    check_walk(sum(-(-c // 256) for c in COUNTS) * -(-n // 256), multiprocessors() // 2)
    rows = sum(COUNTS) + BEHIND
    x, w = integers(rows, k, seed=1), integers(len(COUNTS), *((n, k) if layout == "col" else (k, n)), seed=2)
    y = status_of(grouped.grouped_gemm, x, w, ends_of(COUNTS), w_layout=layout, kernel="pair")
    weight = (lambda e: w[e].double().T) if layout == "col" else (lambda e: w[e].double())
    want = by_group(COUNTS, rows, n, lambda e, lo, hi: x[lo:hi].double() @ weight(e))
    assert torch.equal(y, want.to(torch.bfloat16))


@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("n,k", [(1000, 1000), (1032, 72)])
def test_split_clusters_walk_many_tiles(cuda_device, layout, n, k):
    counts = [c % 130 for c in COUNTS] + [3, 0, 61, 128] * 6
    check_walk(sum(-(-c // 64) for c in counts) * -(-n // 128), multiprocessors() // 2)
    rows = sum(counts) + BEHIND
    x, w = integers(rows, k, seed=1), integers(len(counts), *((n, k) if layout == "col" else (k, n)), seed=2)
    y = status_of(grouped.grouped_gemm, x, w, ends_of(counts), w_layout=layout, kernel="split")
    weight = (lambda e: w[e].double().T) if layout == "col" else (lambda e: w[e].double())
    want = by_group(counts, rows, n, lambda e, lo, hi: x[lo:hi].double() @ weight(e))
    assert torch.equal(y, want.to(torch.bfloat16))


@pytest.mark.parametrize("dtype,accumulate", [(torch.bfloat16, False), (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("n,k", [(1304, 1032), (2056, 520)])
def test_gradients_walk_many_tiles(cuda_device, dtype, accumulate, n, k):
    check_walk(len(COUNTS) * -(-n // 256) * -(-k // 256), multiprocessors() // 2)
    rows = sum(COUNTS) + BEHIND
    dy, x = integers(rows, n, seed=1), integers(rows, k, seed=2)
    dy[-BEHIND:] = float("nan")
    out = torch.full((len(COUNTS), n, k), 3.0, device="cuda") if accumulate else None
    dw = status_of(grouped.grouped_gemm_wgrad, dy, x, ends_of(COUNTS), out, dtype=dtype, accumulate=accumulate,
                   kernel="tcgen05")
    lo = 0
    for e, c in enumerate(COUNTS):
        want = dy[lo:lo + c].double().T @ x[lo:lo + c].double() + (3 if accumulate else 0)
        assert torch.equal(dw[e], want.to(dtype)), e
        lo += c


def test_gradients_of_many_groups_in_several_launches(cuda_device):
    counts = [(37 * e) % 300 if e % 5 else 0 for e in range(600)]
    rows, n, k = sum(counts), 136, 264
    dy, x = integers(rows, n, seed=1), integers(rows, k, seed=2)
    dw = status_of(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), dtype=torch.float32, kernel="tcgen05")
    lo = 0
    for e, c in enumerate(counts):
        assert torch.equal(dw[e], (dy[lo:lo + c].double().T @ x[lo:lo + c].double()).float()), e
        lo += c


def codes_of(*shape, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).cuda()


def scales_of(*shape, seed, low=100, high=150):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(low, high, shape, generator=gen, dtype=torch.uint8).cuda()


def values64(q):
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    pair = torch.stack([q.codes & 15, q.codes >> 4], -1).flatten(-2).long()
    return torch.cat([levels, -levels])[pair] * (2.0 ** (q.scales.double() - 127)).repeat_interleave(32, -1)


MX_KERNELS = [("pair", COUNTS, 192, 256), ("split", [c % 130 for c in COUNTS] + [3, 0, 61, 128] * 6, 64, 128)]


@pytest.mark.parametrize("kernel,counts,tokens,columns", MX_KERNELS, ids=["pair", "split"])
@pytest.mark.parametrize("n,k", [(2568, 2080), (2056, 544)])
def test_mxfp4_walks_many_tiles(cuda_device, kernel, counts, tokens, columns, n, k):
    """Scales of one: sums of multiples of 1/4 below 2^18 are exact."""
    check_walk(sum(-(-c // tokens) for c in counts) * -(-n // columns), multiprocessors() // 2)
    rows = sum(counts) + BEHIND
    ones = lambda *shape: torch.full(shape, 127, dtype=torch.uint8, device="cuda")
    a = MXFP4Tensor(codes_of(rows, k // 2, seed=1), ones(rows, k // 32))
    b = MXFP4Tensor(codes_of(len(counts), n, k // 2, seed=2), ones(len(counts), n, k // 32))
    y = status_of(mxfp4.mxfp4_gemm, a, b, ends_of(counts), kernel=kernel)
    av = values64(a)
    want = by_group(counts, rows, n, lambda e, lo, hi: av[lo:hi] @ values64(MXFP4Tensor(b.codes[e], b.scales[e])).T)
    assert torch.equal(y, want.to(torch.bfloat16))


@pytest.mark.parametrize("kernel,counts,tokens,columns", MX_KERNELS, ids=["pair", "split"])
@pytest.mark.parametrize("k,odd", [(2080, 0), (2080, 5), (1024, 3)])
def test_mxfp4_scales_of_many_tiles(cuda_device, kernel, counts, tokens, columns, k, odd):
    """Each row holds a single one, in a block of its own scale: an output is
    one product of two scales.  odd: scale rows that start at odd addresses."""
    n, rows = 2568, sum(counts) + BEHIND
    a_codes = torch.zeros(rows, k // 2, dtype=torch.uint8, device="cuda")
    at = torch.arange(rows, device="cuda") * 37 % k
    a_codes[torch.arange(rows, device="cuda"), at // 2] = torch.where(at % 2 == 0, 0x02, 0x20).to(torch.uint8)
    a_scales = scales_of(rows, k // 32 + 8, seed=1)[:, odd:odd + k // 32]
    b_scales = scales_of(len(counts), n, k // 32 + 8, seed=2)[..., odd:odd + k // 32]
    b = MXFP4Tensor(torch.full((len(counts), n, k // 2), 0x22, dtype=torch.uint8, device="cuda"), b_scales)
    y = status_of(mxfp4.mxfp4_gemm, MXFP4Tensor(a_codes, a_scales), b, ends_of(counts), kernel=kernel)
    power = lambda s: 2.0 ** (s.double() - 127)
    one = power(a_scales.gather(1, (at // 32)[:, None]))
    want = by_group(counts, rows, n, lambda e, lo, hi: one[lo:hi] * power(b_scales[e].T[at[lo:hi] // 32]))
    assert torch.equal(y, want.to(torch.bfloat16))


# --------------------------------------------- the gradient's tensor-core kernel, by name


def test_gradient_kernel_refuses_rows_off_16_bytes(cuda_device):
    ends = ends_of([2, 2])
    for n, k in ((12, 16), (16, 12)):
        with pytest.raises(_native.KmctsError, match="not_supported"):
            grouped.grouped_gemm_wgrad(integers(4, n, seed=1), integers(4, k, seed=2), ends, kernel="tcgen05")


def test_gradient_kernel_keeps_other_groups_out(cuda_device):
    """Infinities and NaN stay in the gradient of the group that holds them,
    whichever side of its boundaries the stages fall."""
    counts = [20, 0, 37, 130, 6]
    rows, n, k = sum(counts) + 9, 72, 96
    dy, x = integers(rows, n, seed=1), integers(rows, k, seed=2)
    want = [dy[lo:lo + c].double().T @ x[lo:lo + c].double()
            for lo, c in zip(torch.tensor([0] + counts).cumsum(0).tolist(), counts)]
    dy[-9:], x[-9:] = float("nan"), float("inf")
    lo = 0
    for e, c in enumerate(counts):
        bad = x.clone()
        bad[lo:lo + c] = float("inf")
        dw = status_of(grouped.grouped_gemm_wgrad, dy, bad, ends_of(counts), kernel="tcgen05")
        for other in range(len(counts)):
            if other != e or c == 0:
                assert torch.equal(dw[other], want[other].to(torch.bfloat16)), (e, other)
            else:
                assert not dw[other].isfinite().any()
        lo += c


def test_gradient_kernel_accumulates_and_clamps_ends(cuda_device):
    x = integers(200, 64, seed=1)
    ends = torch.tensor([50, 30, 2 ** 31 - 1, -7, 120], dtype=torch.int32, device="cuda")
    main = torch.full((5, 64, 64), 0.5, device="cuda")
    for step in (1, 2):
        status_of(grouped.grouped_gemm_wgrad, x, x, ends, main, accumulate=True, kernel="tcgen05")
        for e, (lo, hi) in enumerate([(0, 50), (50, 50), (50, 200), (200, 200), (200, 200)]):
            assert torch.equal(main[e], (0.5 + step * (x[lo:hi].double().T @ x[lo:hi].double())).float())
