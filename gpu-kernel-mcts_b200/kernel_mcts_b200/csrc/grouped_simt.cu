// CUDA-core kernels of the grouped products, for strides and alignments that
// TMA cannot take.  One CTA walks 64 x 64 output tiles of the groups; each
// output is one FP32 accumulator (FP64 for MXFP4) updated by one FMA per step
// of the contracted dimension in increasing order, rounded once.  Bound by the FP32 units (75
// TFLOP/s on B200 at best); the tensor-core kernels take every aligned call.
#include <type_traits>

#include "grouped_common.cuh"

namespace kmcts {
namespace grouped {
namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

// acc[i][j] += sum over depth of a(row, d) * b(col, d), for the thread's 4 x 4
// outputs (rows ty + 16 i, columns tx + 16 j).
template <typename T, typename LoadA, typename LoadB>
__device__ __forceinline__ void tile_product(T (&acc)[4][4], int rows, int cols, int depth, bool a_depth_inner,
                                             bool b_depth_inner, LoadA a, LoadB b) {
    __shared__ T as[kDepth][kTile + 1];
    __shared__ T bs[kDepth][kTile + 1];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int d0 = 0; d0 < depth; d0 += kDepth) {
        for (int i = threadIdx.x; i < kDepth * kTile; i += kThreads) {
            int d = a_depth_inner ? i % kDepth : i / kTile;
            int r = a_depth_inner ? i / kDepth : i % kTile;
            as[d][r] = r < rows && d0 + d < depth ? a(r, d0 + d) : T(0);
            d = b_depth_inner ? i % kDepth : i / kTile;
            r = b_depth_inner ? i / kDepth : i % kTile;
            bs[d][r] = r < cols && d0 + d < depth ? b(r, d0 + d) : T(0);
        }
        __syncthreads();
        const int steps = min(kDepth, depth - d0);  // no step past the end: 0 * inf must not enter
        for (int d = 0; d < steps; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fma(as[d][ty + 16 * i], bs[d][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
}

__device__ __forceinline__ __nv_bfloat16 rounded(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ __nv_bfloat16 rounded(double v) { return __double2bfloat16(v); }

template <Operand KIND>
__global__ void __launch_bounds__(kThreads) grouped_forward_simt(ForwardArgs p) {
    extern __shared__ int table_smem[];
    const GroupTable table(table_smem, p.groups);
    const int tiles_n = (p.n + kTile - 1) / kTile;
    if (threadIdx.x < 32)
        build_group_table(table, p.ends, p.rows, [&](int rows) { return (rows + kTile - 1) / kTile * tiles_n; });
    __syncthreads();
    auto* y = static_cast<__nv_bfloat16*>(p.y);
    int group = 0;
    for (GridWalk walk(0, table.tiles(), blockIdx.x, gridDim.x); walk.more(); walk.next()) {
        const int t = static_cast<int>(walk.at);
        const int e = group_of_tile(table, t, group);
        const int in_group = t - table.tile[e];
        const int64_t row0 = table.row[e] + in_group / tiles_n * kTile;
        const int col0 = in_group % tiles_n * kTile;
        const int rows = min(kTile, static_cast<int>(table.row[e + 1] - row0));
        const int cols = min(kTile, p.n - col0);
        // MXFP4 values reach 6 * 2^127 and products 2^256: FP64 holds them.
        using Sum = std::conditional_t<KIND == Operand::kMxfp4, double, float>;
        Sum acc[4][4] = {};
        if constexpr (KIND == Operand::kMxfp4) {
            auto* x = static_cast<const uint8_t*>(p.x) + row0 * p.ldx;
            auto* xs = p.x_scales + row0 * p.ldxs;
            auto* w = static_cast<const uint8_t*>(p.w) + e * p.w_stride + col0 * p.ldw;
            auto* ws = p.w_scales + e * p.ws_stride + col0 * p.ldws;
            auto value = [](const uint8_t* codes, const uint8_t* scales, int d) {
                return static_cast<double>(e2m1_value(codes[d / 2] >> (d % 2 * 4))) * e8m0_value(scales[d / 32]);
            };
            tile_product(
                acc, rows, cols, p.k, true, true, [&](int r, int d) { return value(x + r * p.ldx, xs + r * p.ldxs, d); },
                [&](int c, int d) { return value(w + c * p.ldw, ws + c * p.ldws, d); });
        } else {
            auto* x = static_cast<const __nv_bfloat16*>(p.x) + row0 * p.ldx;
            auto* w = static_cast<const __nv_bfloat16*>(p.w) + e * p.w_stride;
            constexpr bool col = KIND == Operand::kBf16Col;
            tile_product(
                acc, rows, cols, p.k, true, col, [&](int r, int d) { return __bfloat162float(x[r * p.ldx + d]); },
                [&](int c, int d) {
                    return __bfloat162float(col ? w[(col0 + c) * p.ldw + d] : w[d * p.ldw + col0 + c]);
                });
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = threadIdx.x / 16 + 16 * i, c = threadIdx.x % 16 + 16 * j;
                if (r < rows && c < cols) y[(row0 + r) * p.ldy + col0 + c] = rounded(acc[i][j]);
            }
    }
    if (p.zero_rest) zero_rest_rows(y, p.ldy, table.rows(), p.rows, p.n, blockIdx.x, gridDim.x);
}

__global__ void __launch_bounds__(kThreads) grouped_wgrad_simt(WgradArgs p) {
    extern __shared__ int table_smem[];
    const GroupTable table(table_smem, p.groups);
    const int tiles_k = (p.k + kTile - 1) / kTile;
    const int per_group = (p.n + kTile - 1) / kTile * tiles_k;
    if (threadIdx.x < 32) build_group_table(table, p.ends, p.rows, [&](int) { return per_group; });
    __syncthreads();
    for (GridWalk walk(0, table.tiles(), blockIdx.x, gridDim.x); walk.more(); walk.next()) {
        const int t = static_cast<int>(walk.at);
        const int e = t / per_group;
        if (p.accumulate && table.row[e + 1] == table.row[e]) continue;  // adds nothing: -0.0 + 0.0 is 0.0
        const int n0 = t % per_group / tiles_k * kTile, k0 = t % tiles_k * kTile;
        const int rows = min(kTile, p.n - n0), cols = min(kTile, p.k - k0);
        const int64_t t0 = table.row[e];
        auto* dy = static_cast<const __nv_bfloat16*>(p.dy) + t0 * p.lddy + n0;
        auto* x = static_cast<const __nv_bfloat16*>(p.x) + t0 * p.ldx + k0;
        float acc[4][4] = {};
        tile_product(
            acc, rows, cols, table.row[e + 1] - table.row[e], false, false,
            [&](int r, int d) { return __bfloat162float(dy[d * p.lddy + r]); },
            [&](int c, int d) { return __bfloat162float(x[d * p.ldx + c]); });
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = threadIdx.x / 16 + 16 * i, c = threadIdx.x % 16 + 16 * j;
                if (r >= rows || c >= cols) continue;
                const int64_t at = e * p.dw_stride + (n0 + r) * p.lddw + k0 + c;
                if (p.fp32) {
                    float* dw = static_cast<float*>(p.dw) + at;
                    *dw = p.accumulate ? *dw + acc[i][j] : acc[i][j];
                } else {
                    static_cast<__nv_bfloat16*>(p.dw)[at] = __float2bfloat16_rn(acc[i][j]);
                }
            }
    }
}

unsigned grid_for(int64_t tiles) {
    const int64_t most = 8LL * multiprocessor_count();
    return static_cast<unsigned>(tiles < 1 ? 1 : tiles < most ? tiles : most);
}

}  // namespace

int launch_forward_simt(const ForwardArgs& a, Operand kind, cudaStream_t stream) {
    // Every group may end in a partly filled tile.
    const int64_t tiles = (static_cast<int64_t>((a.rows + kTile - 1) / kTile) + a.groups) * ((a.n + kTile - 1) / kTile);
    if (tiles > 0x7fffffff) return KMCTS_ENOTSUP;
    const unsigned grid = grid_for(tiles);
    switch (kind) {
        case Operand::kBf16Col:
            grouped_forward_simt<Operand::kBf16Col><<<grid, kThreads, table_bytes(a.groups, false), stream>>>(a);
            break;
        case Operand::kBf16Row:
            grouped_forward_simt<Operand::kBf16Row><<<grid, kThreads, table_bytes(a.groups, false), stream>>>(a);
            break;
        case Operand::kMxfp4:
            grouped_forward_simt<Operand::kMxfp4><<<grid, kThreads, table_bytes(a.groups, false), stream>>>(a);
            break;
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaGetLastError() == cudaSuccess ? KMCTS_OK : KMCTS_EGEMM;
}

int launch_wgrad_simt(const WgradArgs& a, cudaStream_t stream) {
    const int64_t tiles = static_cast<int64_t>(a.groups) * ((a.n + kTile - 1) / kTile) * ((a.k + kTile - 1) / kTile);
    if (tiles > 0x7fffffff) return KMCTS_ENOTSUP;
    grouped_wgrad_simt<<<grid_for(tiles), kThreads, table_bytes(a.groups, false), stream>>>(a);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaGetLastError() == cudaSuccess ? KMCTS_OK : KMCTS_EGEMM;
}

}  // namespace grouped
}  // namespace kmcts
