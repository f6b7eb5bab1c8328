// Inline-PTX building blocks of the grouped products beyond ptx_sm100.cuh:
// three-dimensional tensor copies (the group is the outermost coordinate) and
// block-scaled 4-bit UMMA.
#pragma once

#include "ptx_sm100.cuh"

namespace kmcts {
namespace ptx {

// Programmatic dependent launch.  wait_for_earlier_grids returns once the
// grids before this one in the stream have finished and their writes are
// visible (at once where the launch did not ask for overlap); every access of
// global memory comes after it, and is a plain one: read-only loads (__ldg,
// const __restrict__ parameters) are for data that nothing writes while the
// kernel runs, and the grid before may still be writing it when this one
// starts.  let_next_grid_start allows the next grid's
// blocks onto SMs that have room for them, up to their own wait.
__device__ __forceinline__ void wait_for_earlier_grids() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void let_next_grid_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// With an L2 cache policy (from createpolicy).
__device__ __forceinline__ void tma_load_3d_hint(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t c0,
                                                 int32_t c1, int32_t c2, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
        : "memory");
}

// Completion counted on an mbarrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster_addr,
                                                 int32_t c0, int32_t c1, int32_t c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// With an L2 cache policy (from createpolicy).
__device__ __forceinline__ void tma_store_3d_hint(const CUtensorMap* map, const void* src, int32_t c0, int32_t c1,
                                                  int32_t c2, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%2, %3, %4}], [%1], %5;" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(smem_addr(src)), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
        : "memory");
}

// Adds the box to global memory instead of storing it (one addition per
// element, so the result does not depend on any order).
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, const void* src, int32_t c0, int32_t c1,
                                           int32_t c2) {
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(smem_addr(src)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// Asynchronous 16-byte store into the shared memory of any CTA of the cluster;
// its bytes are counted on an mbarrier of that CTA (both from mapa_shared).
__device__ __forceinline__ void st_async_v4(uint32_t cluster_addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                            uint32_t bar_cluster_addr) {
    asm volatile(
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(cluster_addr),
        "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar_cluster_addr)
        : "memory");
}

// Each of the 32 rows of 16 bytes at `desc` goes to one TMEM lane of four
// consecutive columns at `taddr`, repeated in all four lane quarters.
template <int CTAS>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[tmem] (+)= (A * A's scales) (B * B's scales)^T for E2M1 operands, one
// E8M0 scale for 32 elements of K, 64 elements of K at a time.
template <int CTAS>
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t a_scales, uint32_t b_scales, uint32_t accumulate) {
    if constexpr (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
                d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
                d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
            : "memory");
}

// Instruction descriptor, kind::mxf4: bits 4-5 which bytes of B's scale words
// this step uses (0 or 2); 7-9 A format (1 = E2M1); 10-11 B format; 17-22
// N >> 3; 23 scale format (1 = E8M0); 27-28 M >> 7; 29-30 A's scale bytes;
// 31 zero: 64 elements of K.
__host__ __device__ constexpr uint32_t make_idesc_mxf4(int m, int n, int scale_id) {
    return (static_cast<uint32_t>(scale_id) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (1u << 23) | (static_cast<uint32_t>(m >> 7) << 27) | (static_cast<uint32_t>(scale_id) << 29);
}

// Shared-memory descriptor without swizzle for tmem_copy_scales: groups of 8
// rows of 16 bytes, 128 bytes apart.
__host__ __device__ constexpr uint64_t make_scale_desc(uint32_t smem_byte_addr) {
    return static_cast<uint64_t>((smem_byte_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 32) |
           (1ull << 46);
}

}  // namespace ptx
}  // namespace kmcts
