// How the blocks of a grid share out numbered work: block b of `blocks` takes
// first + b, first + b + blocks, ... below end.  Host code too, so that it can
// be checked without a GPU.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define KMCTS_HD __host__ __device__ __forceinline__
#else
#define KMCTS_HD inline
#endif

namespace kmcts {
namespace grouped {

// 64 bits: rows and tiles are counted in 32 and may come as close to 2^31 as
// 1024, so that a 32-bit sum with the step of a grid (up to eight blocks an
// SM, 1184 on B200) passes it, turns negative and is below the end again.
struct GridWalk {
    int64_t at, end;
    uint32_t step;

    KMCTS_HD GridWalk(int64_t first, int64_t end_, uint32_t block, uint32_t blocks)
        : at(first + block), end(end_), step(blocks) {}
    KMCTS_HD bool more() const { return at < end; }
    KMCTS_HD void next() { at += step; }
};

}  // namespace grouped
}  // namespace kmcts
