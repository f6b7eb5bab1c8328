"""Products grouped by expert on the GPU, against 64-bit products.

Bars:
* integer-valued inputs: every output bit (FP32 sums of small integers are
  exact in any order, and one rounding follows);
* N(0,1) inputs: products of two BF16 values are exact in FP32; a sum of L
  terms in any order, each addition off by at most one FP32 step (2^-23, which
  covers rounding and truncation), is off by at most g = L * 2^-23 * sum |a b|,
  and the rounding to BF16 adds 2^-8 of the value: |y - ref| <= g + 2^-8 (|ref| + g).
"""

from __future__ import annotations

import time
from concurrent.futures import ThreadPoolExecutor
from threading import Thread

import pytest
import torch

from kernel_mcts_b200 import _native, grouped

pytestmark = pytest.mark.gpu

KERNELS = ["auto", "pair", "split", "simt"]
GRADIENT_KERNELS = ["auto", "simt"]

# Row counts by group: empty groups at both ends and between, single rows,
# lengths around the tiles' edges.
COUNTS = {
    "one_row": [1],
    "edges": [0, 1, 127, 0, 128, 129, 15, 16, 17, 0],
    "long": [600, 0, 257, 3],
    "empty": [0, 0, 0],
}
# (N, K): aligned and not, below and across tiles; 77 x 50 has no aligned row.
SIZES = [(64, 64), (136, 200), (520, 328), (33, 264), (1, 8), (77, 50)]


def ends_of(counts):
    return torch.tensor(counts).cumsum(0).to(torch.int32).cuda()


def integers(*shape, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=gen).to(torch.bfloat16).cuda()


def normals(*shape, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(torch.bfloat16).cuda()


def forward64(x, w, counts, layout):
    """The product and the product of magnitudes, zero behind the last group."""
    n = w.shape[1] if layout == "col" else w.shape[2]
    y, mag = (torch.zeros(x.shape[0], n, dtype=torch.float64, device=x.device) for _ in range(2))
    lo = 0
    for e, c in enumerate(counts):
        m = w[e].double().T if layout == "col" else w[e].double()
        y[lo:lo + c] = x[lo:lo + c].double() @ m
        mag[lo:lo + c] = x[lo:lo + c].double().abs() @ m.abs()
        lo += c
    return y, mag


def wgrad64(dy, x, counts):
    out, mag, lo = [], [], 0
    for c in counts:
        d, v = dy[lo:lo + c].double().T, x[lo:lo + c].double()
        out.append(d @ v)
        mag.append(d.abs() @ v.abs())
        lo += c
    return torch.stack(out), torch.stack(mag)


def within(y, ref, mag, length, half_step):
    g = length * 2.0 ** -23 * mag
    return bool(((y.double() - ref).abs() <= g + half_step * (ref.abs() + g)).all())


def checked(call, *args, **kwargs):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = call(*args, status=status, **kwargs)
    torch.cuda.synchronize()
    assert int(status.item()) == 0, f"device status {int(status.item()):#x}"
    return out


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS)
@pytest.mark.parametrize("n,k", SIZES)
def test_forward_integers_bit_exact(cuda_device, kernel, layout, counts, n, k):
    rows = sum(counts) + 5  # five rows behind the last group
    x = integers(rows, k, seed=1)
    w = integers(len(counts), *((n, k) if layout == "col" else (k, n)), seed=2)
    if kernel in ("pair", "split") and (k % 8 or (layout == "row" and n % 8)):
        with pytest.raises(_native.KmctsError, match="not_supported"):  # rows that TMA cannot address
            grouped.grouped_gemm(x, w, ends_of(counts), w_layout=layout, kernel=kernel)
        return
    y = checked(grouped.grouped_gemm, x, w, ends_of(counts), w_layout=layout, kernel=kernel)
    ref, _ = forward64(x, w, counts, layout)
    assert torch.equal(y, ref.to(torch.bfloat16))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("layout", ["col", "row"])
def test_forward_normals_within_bound(cuda_device, kernel, layout):
    counts, n, k = [70, 0, 300, 1], 264, 1000
    x = normals(sum(counts), k, seed=3)
    w = normals(len(counts), *((n, k) if layout == "col" else (k, n)), seed=4)
    y = checked(grouped.grouped_gemm, x, w, ends_of(counts), w_layout=layout, kernel=kernel)
    ref, mag = forward64(x, w, counts, layout)
    assert within(y, ref, mag, k, 2.0 ** -8)


@pytest.mark.parametrize("kernel", KERNELS)
def test_rows_of_other_groups_and_behind_the_last_do_not_enter(cuda_device, kernel):
    """Infinities and NaN in one group's rows, in the weight of an empty group
    and behind the last group stay there."""
    counts, n, k = [20, 0, 37, 130, 6], 72, 96
    x, w = integers(sum(counts) + 9, k, seed=5), integers(5, n, k, seed=6)
    ref, _ = forward64(x, w, counts, "col")
    x[20:57] = float("nan")  # group 2
    x[-9:] = float("inf")
    w[1] = float("nan")
    y = checked(grouped.grouped_gemm, x, w, ends_of(counts), kernel=kernel)
    keep = torch.ones(len(x), dtype=torch.bool)
    keep[20:57] = False
    assert torch.equal(y[keep], ref.to(torch.bfloat16)[keep])
    assert y[20:57].isnan().all()
    dy = integers(len(x), n, seed=7)
    x[20:57] = integers(37, k, seed=8)
    dy[-9:] = float("nan")
    kernel = kernel if kernel in GRADIENT_KERNELS else "auto"
    dw = checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), kernel=kernel)
    assert torch.equal(dw, wgrad64(dy, x, counts)[0].to(torch.bfloat16))
    # One group's NaN stays in its own gradient, whichever side of a boundary it is.
    x[57:187] = float("inf")
    dw = checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), kernel=kernel)
    others = [0, 1, 2, 4]
    assert torch.equal(dw[others], wgrad64(dy, x, counts)[0].to(torch.bfloat16)[others])


@pytest.mark.parametrize("kernel", KERNELS)
def test_out_given_keeps_rows_behind_the_last_group(cuda_device, kernel):
    counts, n, k = [3, 130], 40, 64
    x, w = integers(140, k, seed=1), integers(2, n, k, seed=2)
    wide = torch.full((140, n + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 8:8 + n]
    y = checked(grouped.grouped_gemm, x, w, ends_of(counts), out, kernel=kernel)
    assert y.data_ptr() == out.data_ptr()
    ref, _ = forward64(x, w, counts, "col")
    assert torch.equal(out[:133], ref[:133].to(torch.bfloat16))
    assert (out[133:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 8 + n:] == 7).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("layout", ["col", "row"])
def test_strided_operands(cuda_device, kernel, layout):
    """Rows with gaps, weights inside a larger tensor, and offsets that break
    16-byte alignment (which the CUDA-core kernel then takes)."""
    counts, n, k = [50, 2, 9], 48, 72
    for offset in (8, 3):
        x = integers(61, k + 16, seed=1)[:, offset:offset + k]
        shape = (n, k) if layout == "col" else (k, n)
        w = integers(3, shape[0] + 2, shape[1] + 24, seed=2)[:, 1:1 + shape[0], offset:offset + shape[1]]
        y = checked(grouped.grouped_gemm, x, w, ends_of(counts), w_layout=layout,
                    kernel=kernel if offset == 8 else "auto")
        assert torch.equal(y, forward64(x, w, counts, layout)[0].to(torch.bfloat16))


@pytest.mark.parametrize("kernel", KERNELS)
def test_one_row_of_any_stride(cuda_device, kernel):
    x = integers(16, 1, seed=1).T  # [1, 16] with strides (1, 1)
    w = integers(1, 24, 16, seed=2)
    out = torch.zeros(24, dtype=torch.bfloat16, device="cuda").as_strided((1, 24), (1, 1))
    checked(grouped.grouped_gemm, x, w, ends_of([1]), out, kernel=kernel)
    assert torch.equal(out, forward64(x, w, [1], "col")[0].to(torch.bfloat16))


@pytest.mark.parametrize("kernel", KERNELS)
def test_ends_out_of_order_or_range_are_clamped(cuda_device, kernel):
    n, k = 64, 64
    x, w = integers(200, k, seed=1), integers(5, n, k, seed=2)
    ends = torch.tensor([50, 30, 2 ** 31 - 1, -7, 120], dtype=torch.int32, device="cuda")
    y = checked(grouped.grouped_gemm, x, w, ends, kernel=kernel)
    counts = [50, 0, 150, 0, 0]
    assert torch.equal(y, forward64(x, w, counts, "col")[0].to(torch.bfloat16))
    dw = checked(grouped.grouped_gemm_wgrad, x, x, ends, kernel=kernel if kernel in GRADIENT_KERNELS else "auto")
    assert torch.equal(dw, wgrad64(x, x, counts)[0].to(torch.bfloat16))


def test_many_groups(cuda_device):
    counts = [(7 * e) % 5 for e in range(1024)]
    x, w = integers(sum(counts), 64, seed=1), integers(1024, 24, 64, seed=2)
    y = checked(grouped.grouped_gemm, x, w, ends_of(counts))
    assert torch.equal(y, forward64(x, w, counts, "col")[0].to(torch.bfloat16))
    dw = checked(grouped.grouped_gemm_wgrad, y, x, ends_of(counts), dtype=torch.float32)
    ref, mag = wgrad64(y, x, counts)
    assert within(dw, ref, mag, 5, 2.0 ** -24)


@pytest.mark.parametrize("kernel", GRADIENT_KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS)
@pytest.mark.parametrize("n,k", SIZES)
def test_wgrad_integers_bit_exact(cuda_device, kernel, dtype, counts, n, k):
    rows = sum(counts) + 5
    dy, x = integers(rows, n, seed=1), integers(rows, k, seed=2)
    dw = checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), dtype=dtype, kernel=kernel)
    assert torch.equal(dw, wgrad64(dy, x, counts)[0].to(dtype))


@pytest.mark.parametrize("kernel", GRADIENT_KERNELS)
def test_wgrad_normals_within_bound(cuda_device, kernel):
    counts, n, k = [70, 0, 2000, 1], 136, 264
    dy, x = normals(sum(counts), n, seed=3), normals(sum(counts), k, seed=4)
    for dtype, half in ((torch.bfloat16, 2.0 ** -8), (torch.float32, 2.0 ** -24)):
        dw = checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), dtype=dtype, kernel=kernel)
        assert within(dw, *wgrad64(dy, x, counts), max(counts), half)


@pytest.mark.parametrize("kernel", GRADIENT_KERNELS)
def test_wgrad_accumulates_into_fp32(cuda_device, kernel):
    counts, n, k = [70, 0, 130, 1], 136, 200
    dy, x = integers(sum(counts), n, seed=3), integers(sum(counts), k, seed=4)
    wide = torch.full((4, n + 1, k + 12), 0.5, device="cuda")
    out = wide[:, :n, 4:4 + k]
    ref = wgrad64(dy, x, counts)[0]
    for step in (1, 2):
        dw = checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), out, accumulate=True, kernel=kernel)
        assert dw.data_ptr() == out.data_ptr() and torch.equal(out, (0.5 + step * ref).float())
    checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), out, kernel=kernel)
    assert torch.equal(out, ref.float())
    assert (wide[:, n:] == 0.5).all() and (wide[:, :, :4] == 0.5).all() and (wide[:, :, 4 + k:] == 0.5).all()


def test_linear_gradients(cuda_device):
    """Forward and both gradients through autograd, with an expanded output
    gradient, against the formulas; and the derivative of a scalar against
    differences of it."""
    counts, n, k = [33, 0, 140, 7], 72, 104
    x, w = integers(190, k, seed=1).requires_grad_(), integers(4, n, k, seed=2).requires_grad_()
    ends = ends_of(counts)
    y = grouped.grouped_linear(x, w, ends)
    dy = integers(190, n, seed=3)
    gx, gw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert torch.equal(y, forward64(x.detach(), w.detach(), counts, "col")[0].to(torch.bfloat16))
    assert torch.equal(gx, forward64(dy, w.detach(), counts, "row")[0].to(torch.bfloat16))
    assert torch.equal(gw, wgrad64(dy, x.detach(), counts)[0].to(torch.bfloat16))
    assert (gx[180:] == 0).all()
    gx, gw = torch.autograd.grad(y.sum(), (x, w))  # an expanded gradient
    ones = torch.ones_like(dy)
    assert torch.equal(gx, forward64(ones, w.detach(), counts, "row")[0].to(torch.bfloat16))
    # The loss sum(y * dy) is linear in one entry of x or w, so a difference of
    # two losses with integer inputs is its derivative exactly.
    def loss(xv, wv):
        return forward64(xv, wv, counts, "col")[0].mul(dy.double())[:180].sum()

    gx, gw = torch.autograd.grad(grouped.grouped_linear(x, w, ends), (x, w), dy)
    base = loss(x.detach(), w.detach())
    for r, c in ((0, 0), (40, 103), (179, 5)):
        moved = x.detach().clone()
        moved[r, c] += 1
        assert (loss(moved, w.detach()) - base).to(torch.bfloat16) == gx[r, c]
    for e, i, j in ((0, 0, 0), (2, 71, 103), (3, 9, 50)):
        moved = w.detach().clone()
        moved[e, i, j] += 1
        assert (loss(x.detach(), moved) - base).to(torch.bfloat16) == gw[e, i, j]


def test_linear_gradients_of_a_row_major_weight(cuda_device):
    counts, n, k = [33, 0, 140, 7], 72, 104
    x, w = integers(190, k, seed=1).requires_grad_(), integers(4, k, n, seed=2).requires_grad_()
    y = grouped.grouped_linear(x, w, ends_of(counts), w_layout="row")
    dy = integers(190, n, seed=3)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(y, forward64(x.detach(), w.detach(), counts, "row")[0].to(torch.bfloat16))
    assert torch.equal(gx, forward64(dy, w.detach(), counts, "col")[0].to(torch.bfloat16))
    assert torch.equal(gw, wgrad64(x.detach(), dy, counts)[0].to(torch.bfloat16))


def test_step_as_a_graph(cuda_device):
    """Forward and backward captured together, after the usual warm-up on a
    side stream, and replayed on other data and other groups."""
    n, k = 136, 256
    x, w = integers(300, k, seed=1).requires_grad_(), integers(3, n, k, seed=2).requires_grad_()
    dy, ends = integers(300, n, seed=3), ends_of([100, 150, 50])

    def step():
        y = grouped.grouped_linear(x, w, ends)
        return (y, *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx, gw = step()
    counts = [17, 0, 260]
    with torch.no_grad():
        x.copy_(integers(300, k, seed=4))
        ends.copy_(ends_of(counts))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, forward64(x.detach(), w.detach(), counts, "col")[0].to(torch.bfloat16))
    assert torch.equal(gx, forward64(dy, w.detach(), counts, "row")[0].to(torch.bfloat16))
    assert torch.equal(gw, wgrad64(dy, x.detach(), counts)[0].to(torch.bfloat16))


def test_graph_with_copies_and_a_side_stream(cuda_device):
    """Calls captured behind a fill, a copy and a join with another stream,
    on which a call of its own was captured."""
    counts, n, k = [40, 0, 30], 128, 256
    x, w = integers(70, k, seed=1), integers(3, n, k, seed=2)
    ends, source = torch.zeros(3, dtype=torch.int32, device="cuda"), ends_of(counts)
    out = torch.ones(80, n, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    ref = forward64(x, w, counts, "col")[0].to(torch.bfloat16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ends.copy_(source)
        out.zero_()
        grouped.grouped_gemm(x, w, ends, out[:70])
        side.wait_stream(torch.cuda.current_stream())
        dw = grouped.grouped_gemm_wgrad(out[:70], x, ends, stream=side, dtype=torch.float32)
        y = grouped.grouped_gemm(out[:70], w, ends, w_layout="row")
        torch.cuda.current_stream().wait_stream(side)
        total = y.float().sum() + dw.sum()
    for _ in range(2):
        ends.fill_(-1)
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:70], ref) and (out[70:] == 0).all()
        assert within(dw, *wgrad64(ref, x, counts), 40, 2.0 ** -24)
        y64, mag = forward64(ref, w, counts, "row")
        assert within(y, y64, mag, n, 2.0 ** -8) and total.isfinite()


def test_two_streams_at_once(cuda_device):
    """Calls that overlap on the GPU share nothing."""
    counts, n, k = [700, 30, 300], 512, 1024
    x, w, ends = integers(1030, k, seed=1), integers(3, n, k, seed=2), ends_of(counts)
    few, few_ends = integers(9, k, seed=3), ends_of([4, 0, 5])
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    results = [[], [], []]
    for _ in range(6):
        results[0].append(grouped.grouped_gemm(x, w, ends, stream=streams[0]))
        results[1].append(grouped.grouped_gemm(few, w, few_ends, kernel="split", stream=streams[1]))
        results[2].append(grouped.grouped_gemm_wgrad(x[:, :n], x, ends, stream=streams[2]))
    torch.cuda.synchronize()
    refs = (forward64(x, w, counts, "col")[0].to(torch.bfloat16),
            forward64(few, w, [4, 0, 5], "col")[0].to(torch.bfloat16),
            wgrad64(x[:, :n], x, counts)[0].to(torch.bfloat16))
    for got, ref in zip(results, refs):
        assert all(torch.equal(g, ref) for g in got)


def test_one_weight_for_all_groups(cuda_device):
    """A weight expanded over the groups (stride 0)."""
    counts, n, k = [40, 3, 90], 128, 256
    x, w = integers(133, k, seed=1), integers(1, n, k, seed=2).expand(3, n, k)
    y = checked(grouped.grouped_gemm, x, w, ends_of(counts))
    assert torch.equal(y, forward64(x, w, counts, "col")[0].to(torch.bfloat16))


@pytest.mark.parametrize("kernel", KERNELS)
def test_offsets_past_32_bits(cuda_device, kernel):
    """Rows of x and y, and groups of w, more than 2^31 elements apart."""
    rows, n, k, far = 70, 72, 64, 2 ** 25 + 8
    x_store = torch.zeros(rows * far, dtype=torch.bfloat16, device="cuda")
    y_store = torch.zeros(rows * far, dtype=torch.bfloat16, device="cuda")
    x, y = (t.as_strided((rows, c), (far, 1)) for t, c in ((x_store, k), (y_store, n)))
    x.copy_(integers(rows, k, seed=1))
    w = y_store.as_strided((3, n, k), (2 ** 30 + 2 ** 20, k, 1), 128)  # groups 2^30 apart, clear of y's rows
    w.copy_(integers(3, n, k, seed=2))
    counts = [30, 0, 40]
    ref = forward64(x, w, counts, "col")[0].to(torch.bfloat16)
    checked(grouped.grouped_gemm, x, w.clone() if kernel == "simt" else w, ends_of(counts), y, kernel=kernel)
    assert torch.equal(y, ref)
    gradient = x_store.as_strided((3, n, k), (2 ** 30 + 2 ** 20, k, 1), 128)
    dy = integers(rows, n, seed=3)
    dw_kernel = kernel if kernel in GRADIENT_KERNELS else "auto"
    checked(grouped.grouped_gemm_wgrad, dy, x, ends_of(counts), gradient, kernel=dw_kernel)
    assert torch.equal(gradient, wgrad64(dy, x, counts)[0].to(torch.bfloat16))


def test_only_the_gradients_asked_for_are_computed(cuda_device):
    x, w = integers(8, 16, seed=1), integers(1, 8, 16, seed=2).requires_grad_()
    y = grouped.grouped_linear(x, w, ends_of([8]))
    before = _native.launch_count()
    y.backward(torch.ones_like(y))
    assert _native.launch_count() == before + 1 and w.grad is not None


def test_second_derivatives_are_refused(cuda_device):
    x, w = integers(8, 16, seed=1).requires_grad_(), integers(1, 8, 16, seed=2)
    y = grouped.grouped_linear(x, w, ends_of([8]))
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_calls_in_a_row_see_each_other(cuda_device):
    """A chain of calls that each read what the one before wrote, long enough
    that launches overlap: directly and as a graph."""
    counts, n = [3, 60, 1], 256
    w = torch.zeros(3, n, n, dtype=torch.bfloat16, device="cuda")
    w[:, torch.arange(n), torch.arange(n).roll(1)] = 1  # y[:, j] = x[:, j - 1]
    ends, x = ends_of(counts), integers(64, n, seed=1)
    buffers = [torch.empty_like(x) for _ in range(2)]

    def chain():
        y = x
        for i in range(40):
            kernel = ("pair", "split")[i // 2 % 2]
            y = grouped.grouped_gemm(y, w, ends, buffers[i % 2], kernel=kernel)

    chain()
    assert torch.equal(buffers[1], x.roll(40, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    x.copy_(integers(64, n, seed=2))
    graph.replay()
    graph.replay()
    assert torch.equal(buffers[1], x.roll(40, 1))


def test_side_stream_and_graph_replay(cuda_device):
    counts, n, k = [40, 3, 90], 128, 256
    x, w = integers(sum(counts), k, seed=1), integers(3, n, k, seed=2)
    ends, out = ends_of(counts), torch.empty(sum(counts), n, dtype=torch.bfloat16, device="cuda")
    ref = forward64(x, w, counts, "col")[0].to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = grouped.grouped_gemm(x, w, ends, stream=side)
    dw = grouped.grouped_gemm_wgrad(y, x, ends, stream=side, dtype=torch.float32)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grouped.grouped_gemm(x, w, ends, out)
        dw2 = grouped.grouped_gemm_wgrad(out, x, ends, dtype=torch.float32)
    for counts in ([40, 3, 90], [0, 133, 0], [133, 0, 0]):
        ends.copy_(ends_of(counts))  # the captured kernels read the ends as they are at replay
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, forward64(x, w, counts, "col")[0].to(torch.bfloat16))
        ref, mag = wgrad64(out, x, counts)
        assert within(dw2, ref, mag, 133, 2.0 ** -24)
    assert within(dw, *wgrad64(y, x, [40, 3, 90]), 133, 2.0 ** -24)


def test_repeated_calls_give_the_same_bits(cuda_device):
    counts, n, k = [5, 0, 60, 19], 256, 2048
    x, w, ends = normals(84, k, seed=1), normals(4, n, k, seed=2), ends_of(counts)
    first = grouped.grouped_gemm(x, w, ends)
    grads = grouped.grouped_gemm_wgrad(first, x, ends)
    for _ in range(5):
        assert torch.equal(grouped.grouped_gemm(x, w, ends), first)
        assert torch.equal(grouped.grouped_gemm_wgrad(first, x, ends), grads)


def test_refusals(cuda_device):
    x, w, ends = integers(6, 16), integers(2, 8, 16), ends_of([2, 4])
    for bad in (ends.long(), ends[:, None], torch.zeros(4, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(TypeError, match="ends"):
            grouped.grouped_gemm(x, w, bad)
    with pytest.raises(ValueError, match="ends must be on"):
        grouped.grouped_gemm(x, w, ends.cpu())
    with pytest.raises(ValueError, match="groups"):
        grouped.grouped_gemm(x, w, ends[:1])
    with pytest.raises(ValueError, match="groups"):
        grouped.grouped_gemm(x, w[:0], ends[:0])
    with pytest.raises(ValueError, match="inner dimensions"):
        grouped.grouped_gemm(x, w, ends, w_layout="row")
    with pytest.raises(ValueError, match="shape"):
        grouped.grouped_gemm(x, w, ends, integers(6, 9))
    with pytest.raises(ValueError, match="contiguous"):
        grouped.grouped_gemm(integers(16, 6).T, w, ends)
    with pytest.raises(ValueError, match="overlapping"):
        grouped.grouped_gemm(x[:1].expand(6, 16), w, ends)
    with pytest.raises(ValueError, match="kernel"):
        grouped.grouped_gemm(x, w, ends, kernel="fast")
    with pytest.raises(ValueError, match="kernel"):
        grouped.grouped_gemm_wgrad(x, x, ends, kernel="split")
    with pytest.raises(ValueError, match="status"):
        grouped.grouped_gemm(x, w, ends, status=torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError, match="rows"):
        grouped.grouped_gemm_wgrad(x[:5], x, ends)
    with pytest.raises(ValueError, match="accumulate"):
        grouped.grouped_gemm_wgrad(x, x, ends, accumulate=True)
    with pytest.raises(TypeError, match="gradient"):
        grouped.grouped_gemm_wgrad(x, x, ends, dtype=torch.float16)
    with pytest.raises(ValueError, match="overlapping"):
        grouped.grouped_gemm_wgrad(x, x, ends, torch.empty(16, 16, dtype=torch.bfloat16, device="cuda").expand(2, 16, 16))
    # Shapes with nothing in them.
    assert grouped.grouped_gemm(x[:0], w, ends).shape == (0, 8)
    assert (grouped.grouped_gemm(x[:, :0], w[:, :, :0], ends) == 0).all()
    assert (grouped.grouped_gemm_wgrad(x[:0], x[:0], ends) == 0).all()


def test_threads_on_their_own_streams():
    counts = [5, 0, 130, 9]
    x, w, ends = integers(sum(counts), 136), integers(4, 200, 136, seed=1), ends_of(counts)
    want = forward64(x, w, counts, "col")[0].to(torch.bfloat16)
    torch.cuda.synchronize()

    def work(_):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            ys = [grouped.grouped_gemm(x, w, ends) for _ in range(50)]
        stream.synchronize()
        return all(torch.equal(y, want) for y in ys)

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))


def test_other_threads_run_while_a_launch_waits():
    # The device sleeps while one thread fills its launch queue and waits; this
    # thread must go on.  Its longest pause stays below half of the sleep.
    x, w, ends = integers(4, 64), integers(1, 64, 64, seed=1), ends_of([4])
    out = grouped.grouped_gemm(x, w, ends)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    begin.record()
    torch.cuda._sleep(2_000_000_000)
    end.record()

    def fill():
        for _ in range(4000):
            grouped.grouped_gemm(x, w, ends, out)

    # The clock starts first: the queue is full within one interpreter switch interval.
    thread = Thread(target=fill)
    pause, last = 0.0, time.perf_counter()
    thread.start()
    while thread.is_alive():
        time.sleep(0.001)
        now = time.perf_counter()
        pause, last = max(pause, now - last), now
    thread.join()
    torch.cuda.synchronize()
    assert pause < begin.elapsed_time(end) / 1000 / 2
