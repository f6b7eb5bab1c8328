// Device code shared by the grouped-product kernels: where each group's rows
// and tiles start, and which tile a unit of work is.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grid_walk.h"
#include "grouped_internal.h"

namespace kmcts {
namespace grouped {

// First row and first tile of every group, and one past the last, in shared
// memory (2 x (groups + 1) ints), and where the kernel splits a group's rows
// evenly over its tiles, the rows of one (another groups + 1).
struct GroupTable {
    int* row;
    int* tile;
    int* step;
    int groups;

    __device__ GroupTable(int* smem, int count)
        : row(smem), tile(smem + count + 1), step(smem + 2 * (count + 1)), groups(count) {}
    __device__ int tiles() const { return tile[groups]; }
    __device__ int rows() const { return row[groups]; }
};

constexpr int table_bytes(int groups, bool steps) { return (steps ? 3 : 2) * 4 * (groups + 1); }

// Built by one whole warp: a running maximum of the ends, clamped to the
// rows there are, and a running sum of tiles_of(rows of the group).  Ends out
// of order or out of range thus only make groups empty or short.  ends ==
// nullptr is one group of all rows.  unit > 0: also the rows of a tile, a
// multiple of unit, for groups of max_step rows a tile at most.
template <typename TilesOf>
__device__ __forceinline__ void build_group_table(const GroupTable& t, const int32_t* ends, int rows,
                                                  TilesOf tiles_of, int max_step = 0, int unit = 0) {
    const int lane = threadIdx.x & 31;
    int last_end = 0, last_tile = 0;
    for (int base = 0; base < t.groups; base += 32) {
        const int e = base + lane;
        int end = 0;
        if (e < t.groups) end = ends == nullptr ? rows : min(max(ends[e], 0), rows);
        if (lane == 0) end = max(end, last_end);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d) end = max(end, other);
        }
        int start = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) start = last_end;
        const int mine = e < t.groups ? tiles_of(end - start) : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += other;
        }
        if (e < t.groups) {
            t.row[e] = start;
            if (unit > 0 && end > start) {
                const int each = (end - start - 1) / ((end - start + max_step - 1) / max_step) + 1;
                t.step[e] = (each + unit - 1) / unit * unit;
            }
            t.tile[e] = last_tile + sum - mine;
        }
        last_end = __shfl_sync(0xffffffffu, end, 31);
        last_tile += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
        t.row[t.groups] = last_end;
        t.tile[t.groups] = last_tile;
    }
}

// The first rows alone, of `count` groups from `first` on (row[count] is one
// past the last): for kernels whose groups all have the same number of tiles.
__device__ __forceinline__ void build_group_rows(int* row, const int32_t* ends, int rows, int first, int count) {
    const int lane = threadIdx.x & 31;
    int last_end = 0;
    for (int base = 0; base < first + count; base += 32) {
        const int e = base + lane;
        int end = e < first + count ? min(max(ends[e], 0), rows) : 0;
        if (lane == 0) end = max(end, last_end);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d) end = max(end, other);
        }
        int start = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) start = last_end;
        if (e >= first && e < first + count) row[e - first] = start;
        last_end = __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) row[count] = last_end;
}

// The group that tile `t` belongs to (the one group with tile[e] <= t <
// tile[e + 1]).  A CTA's tiles come in increasing order, so the search goes on
// from the last tile's group; a search from the start cost a tile more than
// the steps that this takes over a whole launch.
__device__ __forceinline__ int group_of_tile(const GroupTable& table, int t, int& last) {
    int e = last;
    while (table.tile[e + 1] <= t) ++e;
    last = e;
    return e;
}

// Zeroes the rows of Y behind the last group, spread over the whole grid.
__device__ __forceinline__ void zero_rest_rows(__nv_bfloat16* y, int64_t ldy, int first, int rows, int n, int block,
                                               int blocks) {
    for (GridWalk r(first, rows, block, blocks); r.more(); r.next())
        for (int c = threadIdx.x; c < n; c += blockDim.x) y[r.at * ldy + c] = __float2bfloat16(0.0f);
}

// E8M0: 2^(s - 127); 0 is the subnormal 2^-127, 255 is NaN.
__device__ __forceinline__ float e8m0_value(uint32_t s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fffffffu : s << 23);
}

// E2M1 codes of the low four bits: sign, two exponent bits, one mantissa bit.
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const uint32_t e = (code >> 1) & 3, m = code & 1;
    const float size = e == 0 ? 0.5f * m : (1.0f + 0.5f * m) * static_cast<float>(1 << (e - 1));
    return (code & 8) ? -size : size;
}

}  // namespace grouped
}  // namespace kmcts
