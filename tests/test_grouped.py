"""Refusals of the expert-layer products that need no GPU: the Python layer's
argument checks and the C entry points' (which return before any launch)."""

from __future__ import annotations

import pytest
import torch

from kernel_mcts_b200 import _launch, _native, grouped, mxfp4

P = 1 << 20  # stands for a device pointer; no call here gets as far as using it


def test_cpu_tensors_and_other_types_are_refused():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16)
    ends = torch.tensor([2, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        grouped.grouped_gemm(x, w, ends)
    with pytest.raises(TypeError, match="bfloat16"):
        grouped.grouped_gemm(x.float(), w, ends)
    with pytest.raises(ValueError, match="CUDA"):
        grouped.grouped_gemm_wgrad(x, x, ends)
    with pytest.raises(ValueError, match="B layout"):
        grouped.grouped_gemm(x, w, ends, w_layout="diagonal")
    with pytest.raises(ValueError, match="multiple of 32"):
        mxfp4.mxfp4_quantize(torch.zeros(2, 33))
    with pytest.raises(ValueError, match="CUDA"):
        mxfp4.mxfp4_quantize(torch.zeros(2, 32))
    with pytest.raises(TypeError):
        mxfp4.mxfp4_quantize(torch.zeros(2, 32, dtype=torch.int32))
    q = mxfp4.MXFP4Tensor(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8))
    assert q.shape == (2, 32)
    with pytest.raises(ValueError, match="CUDA"):
        mxfp4.mxfp4_dequantize(q)
    with pytest.raises(ValueError, match="CUDA"):
        mxfp4.mxfp4_gemm(q, q)


class FakeStream:
    def __init__(self, index):
        self.device = torch.device("cuda", index)


class FakeTensor:
    def __init__(self, index):
        self.index, self.used_by = index, []

    def get_device(self):
        return self.index

    def record_stream(self, stream):
        self.used_by.append(stream)


def test_a_side_stream_runs_the_call_and_marks_every_tensor(monkeypatch):
    here, side = FakeStream(1), FakeStream(1)
    current = [here]

    class OnStream:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            current.append(self.stream)

        def __exit__(self, *exc):
            current.pop()

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: current[-1])
    monkeypatch.setattr(torch.cuda, "stream", OnStream)
    x, out, result = FakeTensor(1), FakeTensor(1), (FakeTensor(1), FakeTensor(1))

    def call(a, b):
        assert (a, b) == (x, 3) and current[-1] is side
        return result

    assert _launch.run_on(side, (x, None, out), call, x, 3) is result
    assert x.used_by == out.used_by == [side] and [t.used_by for t in result] == [[here], [here]]
    assert _launch.run_on(here, (x,), lambda: current[-1]) is here and x.used_by == [side]
    with pytest.raises(ValueError, match="stream is on"):
        _launch.run_on(FakeStream(0), (x,), call)


def test_sizes_beyond_32_bits_are_refused():
    assert _forward(rows=2 ** 31 - 1) == _native.KMCTS_EINVAL


def _forward(**change):
    args = dict(x=P, ldx=64, w=P, w_stride=64 * 32, ldw=64, layout=0, y=P, ldy=32, ends=P, groups=2, rows=4, n=32, k=64,
                flags=0, kernel=0)
    args.update(change)
    return _native.load().kmcts_bf16_grouped_gemm(*args.values(), None, None)


@pytest.mark.parametrize("change", [
    {"x": None}, {"w": None}, {"y": None}, {"ends": None}, {"groups": 0}, {"groups": 1025}, {"rows": -1}, {"n": -1},
    {"k": -1}, {"ldx": 63}, {"ldw": 63}, {"ldy": 31}, {"layout": 2}, {"layout": 1, "ldw": 31}, {"w_stride": -1},
])
def test_c_grouped_gemm_refuses(change):
    assert _forward(**change) == _native.KMCTS_EINVAL


def test_c_calls_with_nothing_to_write_do_nothing():
    lib = _native.load()
    before = _native.launch_count()
    assert _forward(rows=0) == 0 and _forward(n=0) == 0
    assert lib.kmcts_bf16_grouped_wgrad(P, 64, P, 64, P, 0, 64, 0, 0, P, 2, 8, 0, 64, 0, None, None) == 0
    assert lib.kmcts_mxfp4_quantize(P, 0, 32, P, 16, P, 1, 0, 32, None) == 0
    assert lib.kmcts_mxfp4_dequantize(P, 16, P, 1, P, 0, 32, 0, 32, None) == 0
    assert _native.launch_count() == before


@pytest.mark.parametrize("change", [
    {"dy": None}, {"x": None}, {"dw": None}, {"ends": None}, {"groups": 0}, {"lddy": 31}, {"ldx": 63}, {"lddw": 63},
    {"dw_type": 1}, {"accumulate": 1}, {"rows": -1}, {"dw_stride": -1},
])
def test_c_grouped_wgrad_refuses(change):
    args = dict(dy=P, lddy=32, x=P, ldx=64, dw=P, dw_stride=64 * 32, lddw=64, dw_type=0, accumulate=0, ends=P, groups=2,
                rows=4, n=32, k=64, kernel=0)
    args.update(change)
    assert _native.load().kmcts_bf16_grouped_wgrad(*args.values(), None, None) == _native.KMCTS_EINVAL


@pytest.mark.parametrize("change", [{"k": 33}, {"x": None}, {"codes": None}, {"scales": None}, {"type": 3}, {"ldx": 63},
                                    {"ldc": 31}, {"lds": 1}, {"rows": -1}])
def test_c_mxfp4_quantize_and_dequantize_refuse(change):
    args = dict(x=P, type=0, ldx=64, codes=P, ldc=32, scales=P, lds=2, rows=4, k=64)
    args.update(change)
    x, kind, ldx, codes, ldc, scales, lds, rows, k = args.values()
    lib = _native.load()
    assert lib.kmcts_mxfp4_quantize(x, kind, ldx, codes, ldc, scales, lds, rows, k, None) == _native.KMCTS_EINVAL
    assert lib.kmcts_mxfp4_dequantize(codes, ldc, scales, lds, x, kind, ldx, rows, k, None) == _native.KMCTS_EINVAL


@pytest.mark.parametrize("change", [
    {"k": 48}, {"a": None}, {"a_scales": None}, {"b": None}, {"b_scales": None}, {"y": None}, {"lda": 31}, {"ldas": 1},
    {"ldb": 31}, {"ldbs": 1}, {"ldy": 15}, {"groups": 0}, {"ends": None}, {"b_stride": -1}, {"bs_stride": -1}, {"rows": -1},
])
def test_c_mxfp4_gemm_refuses(change):
    args = dict(a=P, lda=32, a_scales=P, ldas=2, b=P, b_stride=16 * 32, ldb=32, b_scales=P, bs_stride=32, ldbs=2, y=P,
                ldy=16, ends=P, groups=2, rows=4, n=16, k=64, flags=0, kernel=0)
    args.update(change)
    assert _native.load().kmcts_mxfp4_gemm(*args.values(), None, None) == _native.KMCTS_EINVAL


@pytest.mark.parametrize("missing", ["codes", "scales"])
def test_mxfp4_results_come_in_pairs(missing):
    out = mxfp4.MXFP4Tensor(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8))
    with pytest.raises(ValueError, match="codes and scales"):
        mxfp4.mxfp4_quantize(torch.zeros(2, 32), out._replace(**{missing: None}))
