// MXFP4 quantisation and its inverse, each one pass over memory and bound by
// HBM: 2 + 17/32 bytes an element either way for BF16.  Nothing is read twice.
//
// Quantising, a thread holds 64 bytes, all its loads under way together: a
// whole block of 32 elements in a 16-bit type, whose largest magnitude then
// needs no other lane and whose addresses cost one calculation, half a block
// in FP32.  16384 x 8192 on B200: 54 us from BF16 (6.3 TB/s), against 110 us
// with 8 elements a thread (three times the instructions); from FP32 a whole
// block a thread took 128 us (128 bytes a lane outrun L1), half a block 91 us.
// Restoring, a thread writes 8 elements at a time, four times (58 us).
#include "grouped_common.cuh"
#include "ptx_grouped.cuh"

namespace kmcts {
namespace {

using grouped::e8m0_value;

constexpr int kThreads = 256;
constexpr int kChunk = 8;  // elements loaded or stored together

template <int TYPE>
struct Element;
template <>
struct Element<KMCTS_TYPE_BF16> {
    using type = __nv_bfloat16;
    // A shift: the conversion instruction shares a unit with the 4-bit
    // conversions, which it kept busy all the time (16384 x 8192: 115 us).
    static __device__ float to_float(type v) {
        return __uint_as_float(static_cast<uint32_t>(__bfloat16_as_ushort(v)) << 16);
    }
    static __device__ type from_float(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Element<KMCTS_TYPE_FP16> {
    using type = __half;
    static __device__ float to_float(type v) { return __half2float(v); }
    static __device__ type from_float(float v) { return __float2half_rn(v); }
};
template <>
struct Element<KMCTS_TYPE_FP32> {
    using type = float;
    static __device__ float to_float(type v) { return v; }
    static __device__ type from_float(float v) { return v; }
};

template <int TYPE>
struct alignas(16) Chunk {
    typename Element<TYPE>::type v[kChunk];
};

// Eight FP32 values to eight E2M1 codes, round to nearest even, saturating at
// 6; the first in the lowest bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t out;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(out)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return out;
}

// Two E2M1 codes (a byte) to two FP16 values, exactly.
__device__ __forceinline__ __half2 e2m1x2_values(uint32_t byte) {
    uint32_t out;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(out) : "r"(byte));
    return *reinterpret_cast<__half2*>(&out);
}

// A thread block takes `rows_per_block` rows of `per_row` pieces (blocks of 32
// or chunks of 8): enough pieces for its threads whatever K is.
struct Place {
    int64_t row;
    unsigned piece;
};

__device__ __forceinline__ Place place_of(unsigned i, int64_t row0, unsigned per_row, unsigned rows_per_block) {
    if (rows_per_block == 1) return {row0, i};
    const unsigned r = i / per_row;
    return {row0 + r, i - r * per_row};
}

// Chunks that a quantising thread holds, and how many threads share a block.
template <int TYPE>
constexpr int kHeld = TYPE == KMCTS_TYPE_FP32 ? 2 : 4;
template <int TYPE>
constexpr int kSharing = 4 / kHeld<TYPE>;

// The block's largest magnitude as FP32 bits; magnitudes compare as integers,
// and a NaN is larger than infinity.  16-bit types compare in pairs.
template <int TYPE>
__device__ __forceinline__ uint32_t largest_bits(const Chunk<TYPE> (&in)[kHeld<TYPE>]) {
    uint32_t m = 0;
    if constexpr (TYPE == KMCTS_TYPE_FP32) {
#pragma unroll
        for (int c = 0; c < kHeld<TYPE>; ++c)
#pragma unroll
            for (int j = 0; j < kChunk; ++j) m = max(m, __float_as_uint(in[c].v[j]) & 0x7fffffffu);
        return max(m, __shfl_xor_sync(3u << (threadIdx.x & 30), m, 1));
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint4 words = *reinterpret_cast<const uint4*>(&in[c]);
            m = __vmaxu2(m, __vmaxu2(__vmaxu2(words.x & 0x7fff7fffu, words.y & 0x7fff7fffu),
                                     __vmaxu2(words.z & 0x7fff7fffu, words.w & 0x7fff7fffu)));
        }
        m = max(m & 0xffffu, m >> 16);
        if constexpr (TYPE == KMCTS_TYPE_BF16) return m << 16;
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
    }
}

template <int TYPE, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
    mxfp4_quantize_kernel(const typename Element<TYPE>::type* x, int64_t ldx, uint8_t* codes, int64_t ldc,
                          uint8_t* scales, int64_t lds, int64_t rows, unsigned per_row, unsigned rows_per_block) {
    ptx::let_next_grid_start();
    ptx::wait_for_earlier_grids();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_per_block;
    const unsigned here = static_cast<unsigned>(min(static_cast<int64_t>(rows_per_block), rows - row0));
    const unsigned total = here * per_row;
    // per_row is even where two threads share a block, so both take the loop
    // together.
    constexpr int kChunks = kHeld<TYPE>;
    for (unsigned i = threadIdx.x; i < total; i += kThreads) {
        const Place at = place_of(i, row0, per_row, rows_per_block);
        const auto* src = x + at.row * ldx + static_cast<int64_t>(at.piece) * (kChunks * kChunk);
        Chunk<TYPE> in[kChunks];
        if constexpr (ALIGNED) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) in[c] = reinterpret_cast<const Chunk<TYPE>*>(src)[c];
        } else {
#pragma unroll
            for (int j = 0; j < kChunks * kChunk; ++j) in[j / kChunk].v[j % kChunk] = src[j];
        }
        // floor(log2) is the exponent field less 127 (a subnormal's is 0, and
        // below the smallest scale either way); E2M1's largest exponent is 2.
        const uint32_t field = largest_bits<TYPE>(in) >> 23;
        const uint32_t scale = field == 255 ? 255 : field > 2 ? field - 2 : 0;
        // 1 / scale = 2^(127 - scale): exact, normal for every scale there is.
        const float inverse = __uint_as_float(scale == 255 ? 0u : (254 - scale) << 23);
        uint32_t packed[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            float v[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk; ++j) v[j] = Element<TYPE>::to_float(in[c].v[j]) * inverse;
            packed[c] = e2m1x8(v);
        }
        uint8_t* dst = codes + at.row * ldc + static_cast<int64_t>(at.piece) * (4 * kChunks);
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int j = 0; j < 4 * kChunks; ++j) dst[j] = static_cast<uint8_t>(packed[j / 4] >> (8 * (j % 4)));
        } else if constexpr (kChunks == 4) {
            *reinterpret_cast<uint4*>(dst) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        } else {
            *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
        }
        if (at.piece % kSharing<TYPE> == 0) scales[at.row * lds + at.piece / kSharing<TYPE>] = static_cast<uint8_t>(scale);
    }
}

// Chunks that a thread of the restoring kernel loads before it works on the
// first: one at a time left HBM more than half idle (16384 x 8192 to BF16
// 141 us, 58 with four).
constexpr int kBatch = 4;

template <int TYPE, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
    mxfp4_dequantize_kernel(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds,
                            typename Element<TYPE>::type* out, int64_t ldo, int64_t rows, unsigned per_row,
                            unsigned rows_per_block) {
    ptx::let_next_grid_start();
    ptx::wait_for_earlier_grids();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_per_block;
    const unsigned here = static_cast<unsigned>(min(static_cast<int64_t>(rows_per_block), rows - row0));
    const unsigned total = here * per_row;
    for (unsigned first = threadIdx.x; first < total; first += kBatch * kThreads) {
        uint32_t packed[kBatch], scale[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned i = first + b * kThreads;
            if (i >= total) break;
            const Place at = place_of(i, row0, per_row, rows_per_block);
            const uint8_t* src = codes + at.row * ldc + static_cast<int64_t>(at.piece) * (kChunk / 2);
            if constexpr (ALIGNED) {
                packed[b] = *reinterpret_cast<const uint32_t*>(src);
            } else {
                packed[b] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) packed[b] |= static_cast<uint32_t>(src[j]) << (8 * j);
            }
            scale[b] = scales[at.row * lds + at.piece / 4];
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned i = first + b * kThreads;
            if (i >= total) break;
            const Place at = place_of(i, row0, per_row, rows_per_block);
            const float s = e8m0_value(scale[b]);
            Chunk<TYPE> values;
#pragma unroll
            for (int j = 0; j < kChunk; j += 2) {
                const float2 pair = __half22float2(e2m1x2_values(packed[b] >> (4 * j) & 0xff));
                values.v[j] = Element<TYPE>::from_float(pair.x * s);
                values.v[j + 1] = Element<TYPE>::from_float(pair.y * s);
            }
            auto* dst = out + at.row * ldo + static_cast<int64_t>(at.piece) * kChunk;
            if constexpr (ALIGNED) {
                *reinterpret_cast<Chunk<TYPE>*>(dst) = values;
            } else {
#pragma unroll
                for (int j = 0; j < kChunk; ++j) dst[j] = values.v[j];
            }
        }
    }
}

bool aligned(const void* p, int64_t stride_bytes, int to) {
    return reinterpret_cast<uintptr_t>(p) % to == 0 && stride_bytes % to == 0;
}

// Rows of a thread block: `each` pieces a thread where there is enough for
// every SM, one where there is not (a few rows: the call is as long as one
// thread's work).
unsigned rows_per_block(int64_t rows, unsigned per_row, int each) {
    const int64_t pieces = rows * per_row;
    const unsigned want = pieces > 8LL * kThreads * multiprocessor_count() ? each * kThreads : kThreads;
    const unsigned fit = want / per_row;
    return fit < 1 ? 1 : fit;
}

template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), int64_t blocks, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[1];
    grouped::allow_early_start(&attr[0]);
    config.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
    config.blockDim = dim3(kThreads, 1, 1);
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (err == cudaSuccess) return KMCTS_OK;
    cudaGetLastError();  // reported here, not by the caller's next call
    return KMCTS_EGEMM;
}

template <int TYPE>
int quantize(const void* X, int64_t ldx, uint8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, int64_t rows,
             int K, cudaStream_t stream) {
    using T = typename Element<TYPE>::type;
    const unsigned per_row = K / 32 * kSharing<TYPE>, per_block = rows_per_block(rows, per_row, 1);
    const int64_t blocks = (rows + per_block - 1) / per_block;
    if (blocks > 0x7fffffff) return KMCTS_EINVAL;
    const bool vec = aligned(X, ldx * sizeof(T), 16) && aligned(codes, ldc, 16);
    return launch(vec ? mxfp4_quantize_kernel<TYPE, true> : mxfp4_quantize_kernel<TYPE, false>, blocks, stream,
                  static_cast<const T*>(X), ldx, codes, ldc, scales, lds, rows, per_row, per_block);
}

template <int TYPE>
int dequantize(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, void* out, int64_t ldo,
               int64_t rows, int K, cudaStream_t stream) {
    using T = typename Element<TYPE>::type;
    const unsigned per_row = K / kChunk, per_block = rows_per_block(rows, per_row, kBatch);
    const int64_t blocks = (rows + per_block - 1) / per_block;
    if (blocks > 0x7fffffff) return KMCTS_EINVAL;
    const bool vec = aligned(out, ldo * sizeof(T), 16) && aligned(codes, ldc, 4);
    return launch(vec ? mxfp4_dequantize_kernel<TYPE, true> : mxfp4_dequantize_kernel<TYPE, false>, blocks, stream,
                  codes, ldc, scales, lds, static_cast<T*>(out), ldo, rows, per_row, per_block);
}

}  // namespace
}  // namespace kmcts

using namespace kmcts;

extern "C" {

int kmcts_mxfp4_quantize(const void* X, int x_type, int64_t ldx, void* codes, int64_t ldc, void* scales, int64_t lds,
                         int64_t rows, int K, void* stream) {
    if (rows < 0 || K < 0 || K % 32 != 0) return KMCTS_EINVAL;
    if (rows == 0 || K == 0) return KMCTS_OK;
    if (!X || !codes || !scales || ldx < K || ldc < K / 2 || lds < K / 32) return KMCTS_EINVAL;
    auto* c = static_cast<uint8_t*>(codes);
    auto* s = static_cast<uint8_t*>(scales);
    auto st = static_cast<cudaStream_t>(stream);
    switch (x_type) {
        case KMCTS_TYPE_BF16: return quantize<KMCTS_TYPE_BF16>(X, ldx, c, ldc, s, lds, rows, K, st);
        case KMCTS_TYPE_FP16: return quantize<KMCTS_TYPE_FP16>(X, ldx, c, ldc, s, lds, rows, K, st);
        case KMCTS_TYPE_FP32: return quantize<KMCTS_TYPE_FP32>(X, ldx, c, ldc, s, lds, rows, K, st);
        default: return KMCTS_EINVAL;
    }
}

int kmcts_mxfp4_dequantize(const void* codes, int64_t ldc, const void* scales, int64_t lds, void* out, int out_type,
                           int64_t ldo, int64_t rows, int K, void* stream) {
    if (rows < 0 || K < 0 || K % 32 != 0) return KMCTS_EINVAL;
    if (rows == 0 || K == 0) return KMCTS_OK;
    if (!codes || !scales || !out || ldo < K || ldc < K / 2 || lds < K / 32) return KMCTS_EINVAL;
    auto* c = static_cast<const uint8_t*>(codes);
    auto* s = static_cast<const uint8_t*>(scales);
    auto st = static_cast<cudaStream_t>(stream);
    switch (out_type) {
        case KMCTS_TYPE_BF16: return dequantize<KMCTS_TYPE_BF16>(c, ldc, s, lds, out, ldo, rows, K, st);
        case KMCTS_TYPE_FP16: return dequantize<KMCTS_TYPE_FP16>(c, ldc, s, lds, out, ldo, rows, K, st);
        case KMCTS_TYPE_FP32: return dequantize<KMCTS_TYPE_FP32>(c, ldc, s, lds, out, ldo, rows, K, st);
        default: return KMCTS_EINVAL;
    }
}

}  // extern "C"
