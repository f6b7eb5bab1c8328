"""MXFP4 quantisation and products on the GPU.

Quantisation is compared bit for bit with a 64-bit restatement of its
definition.  Products: the product of two E2M1 values is exact, a block's scale
is a power of two, and a sum of K terms in any order, each addition off by at
most one FP32 step, is off by at most g = K * 2^-23 * sum |a b|; the rounding to
BF16 adds 2^-8 of the value.  Integer-valued operands are compared bit for bit.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kernel_mcts_b200 import mxfp4
from kernel_mcts_b200.mxfp4 import MXFP4Tensor

pytestmark = pytest.mark.gpu

KERNELS = ["auto", "pair", "split", "simt"]
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize64(x: np.ndarray):
    """(codes, scales) of x [rows, K] in 64 bits; codes unpacked."""
    blocks = x.astype(np.float64).reshape(x.shape[0], -1, 32)
    largest = np.abs(blocks).max(-1)
    with np.errstate(invalid="ignore"):
        exponent = np.frexp(np.where(np.isfinite(largest), largest, 1.0))[1] - 3
    exponent = np.where(largest == 0, -127, np.clip(exponent, -127, 127))
    with np.errstate(invalid="ignore"):
        size = np.abs(blocks) / 2.0 ** exponent[..., None]
    size = np.minimum(size, 6)
    distance = np.abs(size[..., None] - LEVELS)
    # Nearest level; of two equally near, the even code.
    order = distance + np.array([0, 1e-9] * 4)
    codes = np.where(np.isfinite(largest)[..., None], order.argmin(-1), 0) + 8 * np.signbit(blocks)
    scales = np.where(np.isfinite(largest), exponent + 127, 255)
    return codes.reshape(x.shape), scales


def values64(q: MXFP4Tensor) -> torch.Tensor:
    codes = q.codes.view(torch.uint8)
    pair = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    table = torch.tensor([*LEVELS, *(-LEVELS)], dtype=torch.float64, device=codes.device)
    return table[pair] * (2.0 ** (q.scales.view(torch.uint8).double() - 127)).repeat_interleave(32, -1)


def random_pair(*shape, seed=0, low=119, high=135):
    gen = torch.Generator().manual_seed(seed)
    *lead, k = shape
    return MXFP4Tensor(torch.randint(0, 256, (*lead, k // 2), generator=gen, dtype=torch.uint8).cuda(),
                       torch.randint(low, high, (*lead, k // 32), generator=gen, dtype=torch.uint8).cuda())


def check_quantized(x: torch.Tensor, q: MXFP4Tensor):
    codes, scales = quantize64(x.double().cpu().numpy().reshape(-1, x.shape[-1]))
    got = q.codes.cpu().numpy().reshape(len(codes), -1)
    assert np.array_equal(q.scales.cpu().numpy().reshape(scales.shape), scales)
    real = np.repeat(scales != 255, 32, -1)
    unpacked = np.stack([got & 15, got >> 4], -1).reshape(codes.shape)
    assert np.array_equal(unpacked[real], codes[real])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (129, 4096), (1000, 64), (2, 65536 + 32)])
def test_quantize_bit_exact(cuda_device, dtype, rows, k):
    gen = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=gen) * torch.exp(3 * torch.randn(rows, 1, generator=gen))
    x = x.to(dtype).cuda()
    check_quantized(x, mxfp4.mxfp4_quantize(x))


def test_quantize_ties_saturation_and_signs(cuda_device):
    """Every eighth of a step around each border, both signs, in scale 1 (a 4
    to 7.75 in each block), and powers of two as the largest magnitude."""
    values = torch.arange(0, 8, 1 / 16)
    rows = torch.zeros(len(values), 32)
    rows[:, 0] = 7.75
    rows[:, 1], rows[:, 2], rows[:, 3] = values, -values, 5
    check_quantized(rows.cuda(), mxfp4.mxfp4_quantize(rows.cuda()))
    powers = torch.zeros(254, 32)
    powers[:, 5] = 2.0 ** torch.arange(-126, 128).double()
    powers[:, 6] = powers[:, 5] * 0.4375
    check_quantized(powers.cuda(), mxfp4.mxfp4_quantize(powers.cuda()))


def test_quantize_zeros_subnormals_infinities_and_nan(cuda_device):
    x = torch.zeros(8, 64)
    x[1, 3] = 2.0 ** -149
    x[2, 40] = -(2.0 ** -130)
    x[3, 0], x[3, 1] = 2.0 ** -126, 2.0 ** -128
    x[4, 7] = float("inf")
    x[5, 33] = float("nan")
    x[6, 0], x[6, 31] = -float("inf"), float("nan")
    x[7, 0] = torch.finfo(torch.float32).max
    q = mxfp4.mxfp4_quantize(x.cuda())
    check_quantized(x, q)
    back = mxfp4.mxfp4_dequantize(q, dtype=torch.float32).cpu()
    assert back[4, :32].isnan().all() and (back[4, 32:] == 0).all()
    assert back[5, 32:].isnan().all() and back[6, :32].isnan().all() and (back[0] == 0).all()


def test_quantize_strides_shapes_and_out(cuda_device):
    gen = torch.Generator().manual_seed(9)
    wide = torch.randn(40, 200, generator=gen).to(torch.bfloat16).cuda()
    for offset in (8, 3):  # aligned and unaligned rows
        x = wide[:, offset:offset + 160]
        check_quantized(x, mxfp4.mxfp4_quantize(x))
    x = torch.randn(3, 5, 64, generator=gen).cuda()
    q = mxfp4.mxfp4_quantize(x)
    assert q.shape == (3, 5, 64) and q.scales.shape == (3, 5, 2)
    check_quantized(x, q)
    codes = torch.full((15, 40), 99, dtype=torch.uint8, device="cuda")
    scales = torch.full((15, 7), 99, dtype=torch.uint8, device="cuda")
    out = MXFP4Tensor(codes[:, 1:33], scales[:, 2:4])
    mxfp4.mxfp4_quantize(x.view(15, 64), out)
    check_quantized(x.view(15, 64), MXFP4Tensor(out.codes.contiguous(), out.scales.contiguous()))
    assert (codes[:, 0] == 99).all() and (codes[:, 33:] == 99).all()
    assert (scales[:, :2] == 99).all() and (scales[:, 4:] == 99).all()
    assert mxfp4.mxfp4_quantize(x[:0]).shape == (0, 5, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequantize_every_code_and_scale(cuda_device, dtype):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    q = MXFP4Tensor(codes.cuda(), scales.cuda())
    got = mxfp4.mxfp4_dequantize(q, dtype=dtype)
    want = values64(q)
    want[255] = float("nan")
    assert torch.equal(got[:255], want[:255].float().to(dtype)) and got[255].isnan().all()
    wide = torch.full((256, 530), 3.0, dtype=dtype, device="cuda")
    mxfp4.mxfp4_dequantize(q, wide[:, 9:521])
    assert torch.equal(wide[:255, 9:521], got[:255]) and (wide[:, :9] == 3).all() and (wide[:, 521:] == 3).all()


def product64(a, b, counts=None):
    av, bv = values64(a), values64(b)
    if counts is None:
        return av @ bv.T, av.abs() @ bv.T.abs()
    y, mag = (torch.zeros(av.shape[0], bv.shape[1], dtype=torch.float64, device=av.device) for _ in range(2))
    lo = 0
    for e, c in enumerate(counts):
        y[lo:lo + c], mag[lo:lo + c] = av[lo:lo + c] @ bv[e].T, av[lo:lo + c].abs() @ bv[e].abs().T
        lo += c
    return y, mag


def within(y, ref, mag, k):
    g = k * 2.0 ** -23 * mag
    return bool(((y.double() - ref).abs() <= g + 2.0 ** -8 * (ref.abs() + g)).all())


def checked(*args, **kwargs):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = mxfp4.mxfp4_gemm(*args, status=status, **kwargs)
    torch.cuda.synchronize()
    assert int(status.item()) == 0, f"device status {int(status.item()):#x}"
    return out


def ends_of(counts):
    return torch.tensor(counts).cumsum(0).to(torch.int32).cuda()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 32), (1, 300, 64), (17, 129, 96), (130, 128, 256), (200, 264, 544),
                                      (257, 1000, 1024), (500, 77, 2048 + 32)])
def test_product_unit_scales_bit_exact(cuda_device, kernel, rows, n, k):
    """Scales of one: sums of multiples of 1/4 below 2^18 are exact in FP32."""
    a, b = random_pair(rows, k, seed=1, low=127, high=128), random_pair(n, k, seed=2, low=127, high=128)
    y = checked(a, b, kernel=kernel)
    assert torch.equal(y, product64(a, b)[0].to(torch.bfloat16))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("rows,n,k", [(1, 256, 4096), (70, 264, 544), (300, 520, 1056), (256, 512, 512)])
def test_product_random_scales_within_bound(cuda_device, kernel, rows, n, k):
    a, b = random_pair(rows, k, seed=1), random_pair(n, k, seed=2)
    assert within(checked(a, b, kernel=kernel), *product64(a, b), k)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("k", [32, 512, 800, 1024, 2048 + 32 * 15, 3200])
def test_every_block_meets_its_own_scale(cuda_device, kernel, k):
    """One element of 1 in each row, in a block of its own scale: each output
    is one product of two scales, so a scale read from another row or block shows."""
    rows, n = 160, 200
    a_scales = torch.randint(100, 150, (rows, k // 32), generator=torch.Generator().manual_seed(3), dtype=torch.uint8)
    b_scales = torch.randint(100, 150, (n, k // 32), generator=torch.Generator().manual_seed(4), dtype=torch.uint8)
    a_codes, b_codes = torch.zeros(rows, k // 2, dtype=torch.uint8), torch.full((n, k // 2), 0x22, dtype=torch.uint8)
    at = torch.arange(rows) * 37 % k
    a_codes[torch.arange(rows), at // 2] = torch.where(at % 2 == 0, 0x02, 0x20).to(torch.uint8)
    a, b = MXFP4Tensor(a_codes.cuda(), a_scales.cuda()), MXFP4Tensor(b_codes.cuda(), b_scales.cuda())
    y = checked(a, b, kernel=kernel)
    assert torch.equal(y, product64(a, b)[0].to(torch.bfloat16))


@pytest.mark.parametrize("kernel", KERNELS)
def test_extreme_scales(cuda_device, kernel):
    """Scales at the ends of their range whose products are in the middle, and
    products past the range of the result."""
    rows, n, k = 40, 72, 64
    a, b = random_pair(rows, k, seed=1), random_pair(n, k, seed=2)
    for sa, sb in ((0, 254), (254, 0), (1, 253), (20, 230)):
        a.scales.fill_(sa)
        b.scales.fill_(sb)
        assert torch.equal(checked(a, b, kernel=kernel), product64(a, b)[0].to(torch.bfloat16)), (sa, sb)
    a.scales.fill_(254)
    b.scales.fill_(200)
    ref = product64(a, b)[0].to(torch.bfloat16)
    y = checked(a, b, kernel=kernel)
    assert torch.equal(y.isinf(), ref.isinf()) and torch.equal(y, ref)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("counts", [[1], [0, 1, 127, 0, 128, 129, 15, 16, 17, 0], [600, 0, 257, 3], [0, 0]])
@pytest.mark.parametrize("n,k", [(128, 256), (77, 96), (264, 800)])
def test_grouped_product_bit_exact(cuda_device, kernel, counts, n, k):
    rows = sum(counts) + 5
    a = random_pair(rows, k, seed=1, low=127, high=128)
    b = random_pair(len(counts), n, k, seed=2, low=127, high=128)
    y = checked(a, b, ends_of(counts), kernel=kernel)
    assert torch.equal(y, product64(a, b, counts)[0].to(torch.bfloat16))
    out = torch.full((rows, n + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    checked(a, b, ends_of(counts), out[:, :n], kernel=kernel)
    assert torch.equal(out[:sum(counts), :n], y[:sum(counts)]) and (out[sum(counts):] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_scales_stay_in_their_rows(cuda_device, kernel):
    counts, n, k = [20, 37, 70], 136, 352
    a, b = random_pair(130, k, seed=1, low=127, high=128), random_pair(3, n, k, seed=2, low=127, high=128)
    ref = product64(a, b, counts)[0].to(torch.bfloat16)
    a.scales[20:57, 10] = 255  # the last block of group 1's rows
    a.scales[127:] = 255       # behind the last group
    b.scales[2, 5, 3] = 255
    y = checked(a, b, ends_of(counts), kernel=kernel)
    assert torch.equal(y[:20], ref[:20]) and y[20:57].isnan().all()
    assert y[57:127, 5].isnan().all()
    keep = torch.arange(n) != 5
    assert torch.equal(y[57:127][:, keep.cuda()], ref[57:127][:, keep.cuda()]) and (y[127:] == 0).all()


@pytest.mark.parametrize("kernel", KERNELS)
def test_strided_operands(cuda_device, kernel):
    rows, n, k = 70, 136, 320
    for code_at, scale_at in ((16, 8), (16, 3), (5, 0)):
        wide_a, wide_b = random_pair(rows, k + 512, seed=1), random_pair(2, n + 1, k + 512, seed=2)
        a = MXFP4Tensor(wide_a.codes[:, code_at:code_at + k // 2], wide_a.scales[:, scale_at:scale_at + k // 32])
        b = MXFP4Tensor(wide_b.codes[:, 1:, code_at:code_at + k // 2], wide_b.scales[:, 1:, scale_at:scale_at + k // 32])
        y = checked(a, b, ends_of([30, 40]), kernel=kernel if code_at == 16 else "auto")
        assert within(y, *product64(a, b, [30, 40]), k)


def test_torch_types_and_empty_shapes(cuda_device):
    a, b = random_pair(4, 64, seed=1), random_pair(8, 64, seed=2)
    typed = [MXFP4Tensor(t.codes.view(torch.float4_e2m1fn_x2), t.scales.view(torch.float8_e8m0fnu)) for t in (a, b)]
    assert torch.equal(mxfp4.mxfp4_gemm(*typed), mxfp4.mxfp4_gemm(a, b))
    assert mxfp4.mxfp4_gemm(random_pair(0, 64), b).shape == (0, 8)
    assert mxfp4.mxfp4_gemm(a, random_pair(0, 64)).shape == (4, 0)
    assert (mxfp4.mxfp4_gemm(random_pair(4, 0), random_pair(8, 0)) == 0).all()


def test_layer_of_experts_from_bf16(cuda_device):
    """As served: weights quantised once, activations on the way, then the
    grouped product, on a side stream and as a replayed graph."""
    counts, n, k = [9, 0, 130, 1], 264, 512
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(sum(counts), k, generator=gen).to(torch.bfloat16).cuda()
    w = mxfp4.mxfp4_quantize(torch.randn(4, n, k, generator=gen).to(torch.bfloat16).cuda())
    ends = ends_of(counts)
    a = mxfp4.mxfp4_quantize(x)
    y = mxfp4.mxfp4_gemm(a, w, ends)
    assert within(y, *product64(a, w, counts), k)
    restored = mxfp4.mxfp4_dequantize(a, dtype=torch.float32)
    assert torch.equal(restored.double(), values64(a))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y2 = mxfp4.mxfp4_gemm(mxfp4.mxfp4_quantize(x, stream=side), w, ends, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y2, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y3 = mxfp4.mxfp4_gemm(mxfp4.mxfp4_quantize(x), w, ends)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y3, -y)


def test_refusals(cuda_device):
    a, b = random_pair(4, 64), random_pair(8, 64)
    with pytest.raises(ValueError, match="scales must have shape"):
        mxfp4.mxfp4_gemm(MXFP4Tensor(a.codes, a.scales[:, :1]), b)
    with pytest.raises(ValueError, match="inner dimensions"):
        mxfp4.mxfp4_gemm(a, random_pair(8, 96))
    with pytest.raises(ValueError, match="dimensions"):
        mxfp4.mxfp4_gemm(a, b, ends_of([4]))
    with pytest.raises(ValueError, match="groups"):
        mxfp4.mxfp4_gemm(a, random_pair(2, 8, 64), ends_of([4]))
    with pytest.raises(ValueError, match="multiple of 32"):
        mxfp4.mxfp4_gemm(MXFP4Tensor(a.codes[:, :8], a.scales[:, :1]), b)
    with pytest.raises(ValueError, match="shape"):
        mxfp4.mxfp4_dequantize(a, torch.zeros(4, 32, device="cuda"))
    with pytest.raises(TypeError, match="values must be"):
        mxfp4.mxfp4_dequantize(a, dtype=torch.float64)
    with pytest.raises(ValueError, match="two-dimensional or contiguous"):
        mxfp4.mxfp4_quantize(torch.zeros(2, 3, 64, device="cuda").transpose(0, 1))
