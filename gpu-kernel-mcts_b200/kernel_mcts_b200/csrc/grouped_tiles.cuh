// What the tensor-core kernels of the grouped products share: operand kinds,
// tensor maps, failure reporting and the transposed epilogue.
#pragma once

#include "gemm_common.cuh"
#include "grouped_common.cuh"
#include "ptx_grouped.cuh"

namespace kmcts {
namespace grouped {

using gemm::drain_limit;
using gemm::kDefaultWaitNs;
using gemm::kMaxSmem;
using gemm::kRoleDrain;
using gemm::kRoleEpilogue;
using gemm::kRoleMma;
using gemm::kRoleProducer;
using gemm::record_failure;
using gemm::TileCoord;

// The products' operands, by how the MMA's A (the weight; for the weights'
// gradient, the output gradient) lies in memory.
enum class Kind { kCol, kRow, kMxfp4, kWgrad };

// Division by a number known at launch: every role of a kernel finds its next
// tile between two of its waits, and the divide instruction sequences there
// cost 0.3 us a tile (weights' gradient of 16 groups of 512 rows, 4096 x 4096:
// 260 us, 254 us without them; 8192 x 2048 x 512 21.4 and 18.9).
struct Divisor {
    uint32_t d, inverse;  // floor(2^32 / d), at most 2^32 - 1

    __host__ __device__ static constexpr uint32_t inverse_of(uint32_t d) {
        return d <= 1 ? 0xffffffffu : static_cast<uint32_t>((1ull << 32) / d);
    }
    __host__ static Divisor of(uint32_t d) { return {d, inverse_of(d)}; }
    // n / d: the product with the inverse is that or one less.
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
        const uint32_t q = __umulhi(n, inverse);
        return n - q * d >= d ? q + 1 : q;
    }
};

// Divisor::inverse_of(1..7), for a strip of fewer than eight tiles.
static __constant__ uint32_t kInverse[8] = {0, Divisor::inverse_of(1), Divisor::inverse_of(2), Divisor::inverse_of(3),
                                            Divisor::inverse_of(4), Divisor::inverse_of(5), Divisor::inverse_of(6),
                                            Divisor::inverse_of(7)};

// Tile `t` of num_m x num_n: eight tiles down a column strip before moving
// right, so that CTAs at work together share both operands' panels in L2.
// strip is 8 num_n.
__device__ __forceinline__ TileCoord raster(uint32_t t, int num_m, const Divisor& strip) {
    const uint32_t g = strip.quotient(t), r = t - g * strip.d;
    const uint32_t rows = num_m - 8 * g;
    if (rows >= 8) return {static_cast<int>(8 * g + (r & 7)), static_cast<int>(r >> 3)};
    const uint32_t n = Divisor{rows, kInverse[rows]}.quotient(r);
    return {static_cast<int>(8 * g + r - n * rows), static_cast<int>(n)};
}

__host__ __device__ constexpr int round_up(int v, int to) { return (v + to - 1) / to * to; }

// A position in a ring of stages.
template <int STAGES>
struct Ring {
    int stage = 0;
    uint32_t phase = 0;
    __device__ void next() {
        if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
        }
    }
};

// One scale word (four blocks' bytes) of row `r` in the layout that
// tcgen05.cp spreads over TMEM: 32 rows of 16 bytes, row r of 128 in byte
// column 4 (r / 32) of row r % 32.
__device__ __forceinline__ uint32_t scale_word_offset(int r) {
    return static_cast<uint32_t>(r / 128 * 512 + r % 32 * 16 + r % 128 / 32 * 4);
}

// The scales of one operand: no byte outside [begin, end) is read.
struct ScaleSpan {
    const uint8_t* begin;
    const uint8_t* end;
};

// The 16-byte words, aligned, that hold 32 consecutive scale bytes of a row
// from block `first` (a multiple of 32) of `blocks`: two, or three where the
// row starts at an odd address.  A word may reach into other rows of the span;
// what of it lies outside the span reads as zero.  Loads only, so that they can
// be under way while the thread does something else (byte by byte, rows at odd
// addresses took 1269 us for 8192 x 8192 x 8224 where 8192 took 276).
__device__ __forceinline__ void load_scale_words(const uint8_t* row, int first, int blocks, const ScaleSpan& span,
                                                 uint4 (&out)[3]) {
#pragma unroll
    for (int c = 0; c < 3; ++c) out[c] = make_uint4(0, 0, 0, 0);
    if (row == nullptr) return;
    const int offset = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
    const int bytes = offset + min(32, blocks - first);
    const uint8_t* base = row + first - offset;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        if (16 * c >= bytes) break;
        const uint8_t* src = base + 16 * c;
        if (src >= span.begin && src + 16 <= span.end) {
            out[c] = *reinterpret_cast<const uint4*>(src);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < 16; ++b)
                if (src + b >= span.begin && src + b < span.end)
                    w[b / 4] |= static_cast<uint32_t>(src[b]) << (8 * (b % 4));
            out[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// The 32 bytes themselves, from load_scale_words' words; bytes past the row's
// end are zeros (any finite scale serves, the codes there are zeros).
__device__ __forceinline__ void align_scales(const uint8_t* row, int first, int blocks, const uint4 (&words)[3],
                                             uint4 (&out)[2]) {
    const unsigned offset = static_cast<unsigned>(reinterpret_cast<uintptr_t>(row) & 15);
    uint32_t q[12] = {words[0].x, words[0].y, words[0].z, words[0].w, words[1].x, words[1].y,
                      words[1].z, words[1].w, words[2].x, words[2].y, words[2].z, words[2].w};
    if (offset != 0) {
#pragma unroll
        for (int i = 0; i < 10; ++i) q[i] = (offset & 8) ? q[i + 2] : q[i];
#pragma unroll
        for (int i = 0; i < 9; ++i) q[i] = (offset & 4) ? q[i + 1] : q[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = __funnelshift_r(q[i], q[i + 1], 8 * (offset & 3));
    }
    const int left = blocks - first;
    if (left < 32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int valid = left - 4 * i;
            q[i] = valid >= 4 ? q[i] : valid <= 0 ? 0 : q[i] & ((1u << (8 * valid)) - 1);
        }
    }
    out[0] = make_uint4(q[0], q[1], q[2], q[3]);
    out[1] = make_uint4(q[4], q[5], q[6], q[7]);
}

// 32 TMEM lanes x 32 columns in the registers of 8 x 8 matrices: after it, r[16
// h + 4 t + 2 g + i] is lane 16 h + 8 g + l / 4, column 8 t + 2 (l % 4) + i, for
// thread l of the warp.
__device__ __forceinline__ void load_rows_of_8(uint32_t taddr, uint32_t (&r)[32]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t* q = r + 16 * h;
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
              "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15])
            : "r"(taddr + (static_cast<uint32_t>(16 * h) << 16)));
    }
    ptx::tmem_wait_ld();
}

// Writes a 32-token chunk of an accumulator whose lanes are output columns
// (from load_rows_of_8): lane l is column col0 + l of tokens 0..31.  The values
// turn round in a 32 x 64-byte staging buffer of the warp's own, four 8 x 8
// matrices at a time, so that four threads write 64 consecutive bytes of one
// token's row.  Chunk j of token t's 64 bytes stands at j ^ (t / 2) % 4: no two
// rows of a matrix share banks.
__device__ __forceinline__ void store_transposed(const uint32_t (&r)[32], uint8_t* staging, __nv_bfloat16* y,
                                                 int64_t ldy, int tokens, int col0, int n, bool vec, int lane) {
    __syncwarp();  // the chunk before has been read
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int token = 8 * t + lane % 8;
        const uint32_t at = ptx::smem_addr(staging + token * 64 + ((lane / 8) ^ (token / 2 % 4)) * 16);
        asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at),
                     "r"(gemm::pack_bf16x2(r[4 * t], r[4 * t + 1])), "r"(gemm::pack_bf16x2(r[4 * t + 2], r[4 * t + 3])),
                     "r"(gemm::pack_bf16x2(r[16 + 4 * t], r[16 + 4 * t + 1])),
                     "r"(gemm::pack_bf16x2(r[16 + 4 * t + 2], r[16 + 4 * t + 3]))
                     : "memory");
    }
    __syncwarp();
    if (!vec) {
        // Rows at any alignment: 32 threads write 64 consecutive bytes, two
        // each (16 experts, 8192 rows, 4095 x 4096: 307 us with eight
        // two-byte stores for each 16 bytes, 231 so).
        if (col0 + lane < n)
            for (int j = 0; j < min(tokens, 32); ++j)
                y[j * ldy + col0 + lane] = *reinterpret_cast<const __nv_bfloat16*>(
                    staging + j * 64 + ((lane / 8) ^ (j / 2 % 4)) * 16 + lane % 8 * 2);
        return;
    }
    const int col = col0 + lane % 4 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = i * 8 + lane / 4;
        if (j >= tokens || col >= n) continue;
        __nv_bfloat16* dst = y + j * ldy + col;
        const auto* src = reinterpret_cast<const __nv_bfloat16*>(staging + j * 64 + (lane % 4 ^ (j / 2 % 4)) * 16);
        if (col + 8 <= n) {
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
        } else {
            for (int b = 0; b < 8 && col + b < n; ++b) dst[b] = src[b];
        }
    }
}

// Host: a tensor map of `rank` dimensions (dims[0] innermost, strides in bytes
// of dims 1..rank-1).  False where the driver refuses it (alignment).
bool encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims,
                const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle);

// Host: the weight's map (128 rows of 128 bytes, or for kBf16Row two boxes of
// 64 x 64) and three of the tokens', by rows of a box.
bool encode_forward_maps(const ForwardArgs& f, Operand operand, CUtensorMap* w, CUtensorMap (&x)[3],
                         const uint32_t (&box_rows)[3]);

// Host: where the scales of the tokens and of the weights lie.
void scale_spans(const ForwardArgs& f, ScaleSpan* x, ScaleSpan* w);

}  // namespace grouped
}  // namespace kmcts
