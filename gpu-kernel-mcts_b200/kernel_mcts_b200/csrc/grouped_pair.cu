// Grouped products on CTA pairs: one tcgen05.mma.cta_group::2 computes 256
// weight rows x up to 256 tokens (192 in MXFP4) across a cluster of two CTAs.
//
// The weight is the MMA's A and the tokens its B, the accumulator is the
// output transposed: the ragged dimension is then the MMA's N, which an
// instruction descriptor sets at run time in steps of 32, so a group of 70
// tokens costs 96 columns, where tokens in the MMA's rows would cost 256.  A
// group's tokens split evenly over its tiles.  The epilogue turns each chunk
// round in shared memory and writes the valid tokens only.
//
// The weights' gradient (Kind::kWgrad) is the same pipeline with the output
// gradient's columns as A, the input's as B, both MN-major, and the group's
// rows as the contracted dimension.  Its last stage of 128 rows may reach into
// the next group: a warp of each CTA zeroes the foreign rows of the last
// 16-row step in shared memory (both operands: 0 * inf is not 0), and the MMA
// takes no further step.
//
// Roles per CTA: warp 0 TMA producer; warp 1 MMA (the pair's leader issues);
// warps 2-9 epilogue; MXFP4 adds four warps that fetch scales and one that
// issues their copies into TMEM, the gradient one that zeroes tails.  Every CTA
// reads the groups' ends itself and walks the tiles round-robin; nothing is
// decided on the host.  Every wait is bounded.
//
// Bounds, measured on two B200 in bursts (graph replays of several calls on
// operands beyond L2; times elsewhere in this file are taken so, too, before
// and after the choice at hand).  8192 rows of 4096 x 4096, PFLOP/s: forward
// products 1.50 to 1.57 with one group, 1.37 to 1.44 with 16 equal ones, 1.22
// to 1.29 with skewed ones; gradients 1.36 to 1.40, 1.13 to 1.19, 1.07 to 1.13;
// MXFP4 at 8192^3 3.75 to 4.06.  The tensor pipe is busy 78% of the time, held
// back by operands from L2 (10 TB/s into the SMs; an MXFP4 tile moves 448 rows
// of them for 256 x 192 outputs).  Skewed groups' tiles differ in width, and
// round-robin leaves the longest pair 8 to 12% over an even share (simulated
// over 40 draws; a shared counter would leave 6%, the widest first 4%).  A
// product of fewer than 74 tiles leaves pairs idle, and a gradient's
// contraction is not split: one tile of 8192 rows takes 42 us.  Gradients of a
// few rows are bound by writing them.
#include <mutex>

#include "grouped_tiles.cuh"

namespace kmcts {
namespace grouped {
namespace {

constexpr int kAccCols = 256;      // TMEM columns from one accumulator to the next (MXFP4: 192)
constexpr int kEpilogueWarps = 8;  // two for each quarter of the TMEM lanes
constexpr int kBaseThreads = 64 + 32 * kEpilogueWarps;
constexpr int kExtraWarp = kBaseThreads / 32;

template <Kind KIND>
struct Pair {
    static constexpr bool kMx = KIND == Kind::kMxfp4;
    static constexpr bool kGrad = KIND == Kind::kWgrad;
    static constexpr bool kAMn = KIND == Kind::kRow || kGrad;  // A (and for the gradient B) MN-major
    static constexpr int kThreads = kBaseThreads + (kMx ? 160 : kGrad ? 32 : 0);
    // K elements of a stage: a block (256 in MXFP4, 64 in BF16: 128 bytes of
    // a K-major row), or two.  BF16 forward products with six stages of one
    // block took 3 to 8% longer than with three of two (16 experts, 8192 rows,
    // 4096 x 4096: 236 us against 228), gradients with five of one 7 to 17%
    // (16 groups of 512 rows: 252 us against 234, one of 8192: 234 against 200).
    // MXFP4 products with three of two, the scales taking turns in two TMEM
    // slots, gained 3% at 8192 x 8192 x 8192 and lost 4 to 5% on grouped and
    // short ones.
    static constexpr int kBlocks = kMx ? 1 : 2;
    static constexpr int kBK = kMx ? 256 : 64 * kBlocks;
    static constexpr int kMaxWidth = kMx ? 192 : 256;
    static constexpr int kABlock = 128 * 128;  // bytes of one block, B's for the widest tile
    static constexpr int kBBlock = kMaxWidth / 2 * 128;
    static constexpr int kABytes = kABlock * kBlocks;
    static constexpr int kBBytes = kBBlock * kBlocks;
    // Scales of a stage: two words a row, of 128 weight rows and 256 tokens.
    static constexpr int kScaleBytes = kMx ? 2 * 512 + 2 * 1024 : 0;
    static constexpr int kStageBytes = kABytes + kBBytes + kScaleBytes;
    // MXFP4: each stage's scales have TMEM columns of their own, 8 + 16.
    static constexpr int kStages = kMx ? 5 : 3;
    static constexpr int kScaleCols = 24;
    static constexpr int kStagingBytes = kGrad ? 4096 : 2048;  // an epilogue warp's
    static constexpr int kStagingOffset = kStages * kStageBytes;
    static constexpr int kBarrierOffset = kStagingOffset + kEpilogueWarps * kStagingBytes;
    static constexpr int kTableOffset = kBarrierOffset + 512;
    // The gradient's table holds first rows only, and of so many groups a launch.
    static constexpr int kMaxGroups = kGrad ? 256 : KMCTS_MAX_GROUPS;
    static constexpr int smem_bytes(int groups) {
        return 1024 + kTableOffset + (kGrad ? 4 * (groups + 1) : table_bytes(groups, true));
    }
    static_assert(2 * kMaxWidth + (kMx ? kStages * kScaleCols : 0) <= 512, "TMEM columns");
    static_assert(smem_bytes(kMaxGroups) <= kMaxSmem, "shared memory");
};

struct PairParams {
    const int32_t* ends;
    int groups, rows;
    int first_group;    // gradient: of this launch
    int n, k;           // the weight is n x k (MMA: n in A's rows; gradient: k in B's columns)
    __nv_bfloat16* y;   // forward output
    int64_t ldy;
    bool vec;           // y rows take 16-byte stores
    bool zero_rest;
    bool fp32, accumulate;  // gradient
    bool stream_out;        // gradient: larger than half of L2
    const uint8_t* x_scales;
    int64_t ldxs;
    const uint8_t* w_scales;
    int64_t ws_stride, ldws;
    ScaleSpan x_span, w_span;
    Divisor strip;      // eight rows of tiles
    Divisor per_group;  // gradient: tiles of a group
    uint64_t limit_ns;
    int* status;
};

// One tile: A rows from n0, B columns (tokens, or columns of the gradient)
// from b0, `width` of them computed and `valid` stored, over `blocks` stages.
struct Tile {
    int e, n0, b0, width, valid, blocks;
    int t0, tail;  // gradient: first contracted row, rows of the last stage (0: full)
};

template <Kind KIND>
__device__ __forceinline__ Tile tile_at(const GroupTable& table, const PairParams& p, int t, int& group) {
    using L = Pair<KIND>;
    Tile out = {};
    if constexpr (L::kGrad) {
        out.e = static_cast<int>(p.per_group.quotient(t));
    } else {
        out.e = group_of_tile(table, t, group);
    }
    const int first = table.row[out.e], rows = table.row[out.e + 1] - first;
    if constexpr (L::kGrad) {
        const TileCoord tc = raster(t - out.e * p.per_group.d, (p.n + 255) / 256, p.strip);
        out.n0 = tc.m_blk * 256;
        out.b0 = tc.n_blk * L::kMaxWidth;
        out.valid = min(L::kMaxWidth, p.k - out.b0);
        out.blocks = (rows + L::kBK - 1) / L::kBK;
        out.t0 = first;
        out.tail = rows % L::kBK;
    } else {
        const int tiles_t = (rows + L::kMaxWidth - 1) / L::kMaxWidth;
        const int step = table.step[out.e];
        const TileCoord tc = raster(t - table.tile[out.e], tiles_t, p.strip);
        out.n0 = tc.n_blk * 256;
        out.b0 = first + tc.m_blk * step;
        out.valid = min(step, first + rows - out.b0);
        out.blocks = (p.k + L::kBK - 1) / L::kBK;
    }
    out.width = round_up(out.valid, 32);
    return out;
}

struct Barriers {
    uint64_t *full, *empty;            // a stage's operands are here; its MMAs are done
    uint64_t *tmem_full, *tmem_empty;  // an accumulator is complete; it has been read
    uint64_t* drain;                   // every MMA is done
    uint64_t *landed, *fixed;          // gradient: a ragged stage is here; its tail is zeroed
    uint64_t *copied, *copies_done;    // MXFP4: a stage's scales are in TMEM; all of them are
};

template <Kind KIND>
__global__ void __launch_bounds__(Pair<KIND>::kThreads, 1)
    grouped_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b128,
                        const __grid_constant__ CUtensorMap map_b64, const __grid_constant__ CUtensorMap map_b32,
                        const __grid_constant__ CUtensorMap map_c, const __grid_constant__ PairParams p) {
    using L = Pair<KIND>;
    constexpr int S = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarrierOffset);
    const Barriers bar = {bars,
                          bars + S,
                          bars + 2 * S,
                          bars + 2 * S + 2,
                          bars + 2 * S + 4,
                          bars + 2 * S + 5,
                          bars + 3 * S + 5,
                          bars + 4 * S + 5,
                          bars + 5 * S + 5};
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 5 * S + 6);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* no_abort = abort + 1;
    int* table_smem = reinterpret_cast<int*>(smem + L::kTableOffset);
    const GroupTable table(table_smem, p.groups);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = static_cast<int>(ptx::cluster_ctarank());
    const bool leader = rank == 0;
    const int first_tile = blockIdx.x / 2, tile_step = gridDim.x / 2;

    ptx::let_next_grid_start();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            // MXFP4: besides the leader's byte count, four scale warps of each CTA.
            ptx::mbar_init(&bar.full[s], L::kMx ? 9 : 1);
            ptx::mbar_init(&bar.empty[s], 1);
            ptx::mbar_init(&bar.landed[s], 1);
            ptx::mbar_init(&bar.fixed[s], 2);
            ptx::mbar_init(&bar.copied[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(&bar.tmem_full[a], 1);
            ptx::mbar_init(&bar.tmem_empty[a], 2 * kEpilogueWarps);
        }
        ptx::mbar_init(bar.drain, 1);
        ptx::mbar_init(bar.copies_done, 1);
        *abort = 0;
        *no_abort = 0;
        ptx::fence_mbarrier_init();
        ptx::prefetch_tensormap(&map_a);
        ptx::prefetch_tensormap(&map_b64);
        if constexpr (L::kGrad) {
            ptx::prefetch_tensormap(&map_c);
        } else {
            ptx::prefetch_tensormap(&map_b128);
            ptx::prefetch_tensormap(&map_b32);
        }
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(tmem_slot, 512);
        ptx::tmem_relinquish_pair();
    }
    // Up to here the launch overlaps the end of the grid before.
    ptx::wait_for_earlier_grids();
    if (warp == 2) {
        if constexpr (L::kGrad) {
            build_group_rows(table.row, p.ends, p.rows, p.first_group, p.groups);
        } else {
            const int tiles_a = (p.n + 255) / 256;
            build_group_table(table, p.ends, p.rows,
                              [&](int rows) { return (rows + L::kMaxWidth - 1) / L::kMaxWidth * tiles_a; }, L::kMaxWidth,
                              32);
        }
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();  // the leader's barriers exist before the peer signals them
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int tiles = L::kGrad ? p.groups * static_cast<int>(p.per_group.d) : table.tiles();
    int group = 0;  // the last tile's
    constexpr int kAccStep = L::kMx ? 192 : kAccCols;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            Ring<S> ring;
            uint32_t issued = 0, issued_phase = 0;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += tile_step) {
                const Tile w = tile_at<KIND>(table, p, t, group);
                const int half = w.width / 2;
                const int a0 = w.n0 + rank * 128, b0 = w.b0 + rank * half;
                // MN-major operands come in boxes of 64 columns, tokens in one
                // box of the next size up (16 experts of 448 tokens, 4096 x
                // 4096: several boxes of 32 rows took 238 us, one box 205).
                const int boxes = (half + 63) / 64;
                const CUtensorMap* mb = half > 64 ? &map_b128 : half > 32 ? &map_b64 : &map_b32;
                const int box_rows = half > 64 ? L::kMaxWidth / 2 : half > 32 ? 64 : 32;
                const uint32_t b_bytes = static_cast<uint32_t>(L::kGrad ? boxes * 8192 : box_rows * 128);  // of a block
                for (int kb = 0; kb < w.blocks; ++kb) {
                    if (!ptx::mbar_wait(&bar.empty[ring.stage], ring.phase ^ 1u, p.limit_ns, abort)) {
                        record_failure(p.status, abort, kRoleProducer);
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + ring.stage * L::kStageBytes;
                    uint8_t* sb = sa + L::kABytes;
                    uint32_t full = ptx::mapa_shared(ptx::smem_addr(&bar.full[ring.stage]), 0);
                    if constexpr (L::kGrad) {
                        // A ragged last stage lands on this CTA's own barrier:
                        // its tail is zeroed before the leader hears of it.
                        int here = L::kBlocks;
                        if (w.tail != 0 && kb == w.blocks - 1) {
                            here = (w.tail + 63) / 64;
                            ptx::mbar_arrive_expect_tx(&bar.landed[ring.stage], here * (L::kABlock + b_bytes));
                            if (leader) ptx::mbar_arrive(&bar.full[ring.stage]);
                            full = ptx::mapa_shared(ptx::smem_addr(&bar.landed[ring.stage]), rank);
                        } else if (leader) {
                            ptx::mbar_arrive_expect_tx(&bar.full[ring.stage], 2 * here * (L::kABlock + b_bytes));
                        }
                        for (int h = 0; h < here; ++h) {
                            const int t0 = w.t0 + kb * L::kBK + h * 64;
                            for (int i = 0; i < 2; ++i)
                                ptx::tma_load_2d_pair(sa + h * L::kABlock + i * 8192, &map_a, full, a0 + 64 * i, t0);
                            for (int i = 0; i < boxes; ++i)
                                ptx::tma_load_2d_pair(sb + h * L::kBBlock + i * 8192, &map_b64, full, b0 + 64 * i, t0);
                        }
                    } else {
                        if (leader) ptx::mbar_arrive_expect_tx(&bar.full[ring.stage], 2 * L::kBlocks * (L::kABlock + b_bytes));
                        for (int h = 0; h < L::kBlocks; ++h) {
                            const int k0 = L::kMx ? kb * 128 : kb * L::kBK + h * 64;  // MXFP4 maps count bytes
                            if constexpr (L::kAMn) {
                                for (int i = 0; i < 2; ++i)
                                    ptx::tma_load_3d_pair(sa + h * L::kABlock + i * 8192, &map_a, full, a0 + 64 * i, k0,
                                                          w.e);
                            } else {
                                ptx::tma_load_3d_pair(sa + h * L::kABlock, &map_a, full, k0, a0, w.e);
                            }
                            ptx::tma_load_2d_pair(sb + h * L::kBBlock, mb, full, k0, b0);
                        }
                    }
                    issued |= 1u << ring.stage;
                    issued_phase = (issued_phase & ~(1u << ring.stage)) | (ring.phase << ring.stage);
                    ring.next();
                }
            }
            // The leader's full barriers count both CTAs' copies; none may be
            // in flight when a CTA leaves.  (A ragged stage's are waited for by
            // the warp that zeroes its tail.)
            for (int s = 0; s < S; ++s) {
                if (leader && (issued & (1u << s)) &&
                    !ptx::mbar_wait(&bar.full[s], (issued_phase >> s) & 1u, drain_limit(p.limit_ns), no_abort))
                    record_failure(p.status, abort, kRoleDrain);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ----------------------------------------------------------------- MMA
        if (lane == 0 && leader) {
            Ring<S> ring;
            uint32_t fixed_phase = 0;  // a bit per stage
            int local = 0;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += tile_step) {
                const Tile w = tile_at<KIND>(table, p, t, group);
                if (w.blocks == 0) continue;
                const int acc = local & 1;
                if (!ptx::mbar_wait(&bar.tmem_empty[acc], ((local >> 1) & 1) ^ 1u, p.limit_ns, abort)) {
                    record_failure(p.status, abort, kRoleMma);
                    break;
                }
                ++local;
                ptx::tc_fence_after();
                const uint32_t d = tmem_base + acc * kAccStep;
                const uint32_t idesc = L::kMx ? ptx::make_idesc_mxf4(256, w.width, 0)
                                              : ptx::make_idesc_bf16_ab(256, w.width, L::kAMn, L::kGrad);
                for (int kb = 0; kb < w.blocks; ++kb) {
                    // MXFP4: the scales' copy has waited for the whole stage.
                    bool here = ptx::mbar_wait(L::kMx ? &bar.copied[ring.stage] : &bar.full[ring.stage], ring.phase,
                                               p.limit_ns, abort);
                    int steps = 4 * L::kBlocks;
                    if constexpr (L::kGrad) {
                        if (here && w.tail != 0 && kb == w.blocks - 1) {
                            here = ptx::mbar_wait_cluster(&bar.fixed[ring.stage], (fixed_phase >> ring.stage) & 1u,
                                                          p.limit_ns, abort);
                            fixed_phase ^= 1u << ring.stage;
                            steps = (w.tail + 15) / 16;
                        }
                    }
                    if (!here) {
                        record_failure(p.status, abort, kRoleMma);
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t sa = ptx::smem_addr(smem + ring.stage * L::kStageBytes);
                    const uint32_t sb = sa + L::kABytes;
                    if constexpr (L::kMx) {
                        const uint32_t ts = tmem_base + 2 * kAccStep + ring.stage * L::kScaleCols;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const uint32_t id = static_cast<uint32_t>(kk % 2 * 2);
                            ptx::umma_mxf4<2>(d, ptx::make_sw128_desc(sa + kk * 32, 16, 1024),
                                              ptx::make_sw128_desc(sb + kk * 32, 16, 1024), idesc | id << 4 | id << 29,
                                              ts + 4 * (kk / 2), ts + 8 + 8 * (kk / 2), (kb | kk) != 0);
                        }
                    } else {
                        for (int kk = 0; kk < steps; ++kk) {
                            const uint32_t a = sa + kk / 4 * L::kABlock, b = sb + kk / 4 * L::kBBlock;
                            const uint64_t adesc = L::kAMn ? ptx::make_sw128_desc(a + kk % 4 * 2048, 8192, 1024)
                                                           : ptx::make_sw128_desc(a + kk % 4 * 32, 16, 1024);
                            const uint64_t bdesc = L::kGrad ? ptx::make_sw128_desc(b + kk % 4 * 2048, 8192, 1024)
                                                            : ptx::make_sw128_desc(b + kk % 4 * 32, 16, 1024);
                            ptx::umma_bf16_pair(d, adesc, bdesc, idesc, (kb | kk) != 0);
                        }
                    }
                    ptx::umma_commit_pair(&bar.empty[ring.stage], 3);
                    ring.next();
                }
                if (ok) ptx::umma_commit_pair(&bar.tmem_full[acc], 3);
            }
            ptx::umma_commit_pair(bar.drain, 3);
        }
        __syncwarp();
    } else if (warp < kExtraWarp) {
        // ------------------------------------------------------------ epilogue
        // Two warps share a quarter's lanes and take its chunks of columns in
        // turn.  (With one warp a quarter the epilogue was longer than the
        // MMAs of a short contraction: 16 x 4096 x 4096 from 64 rows a group
        // took 148 us, the weights' gradient of 512 rows a group 267.)
        const int quarter = warp % 4, turn = (warp - 2) / 4;
        uint8_t* staging = smem + L::kStagingOffset + (warp - 2) * L::kStagingBytes;
        int local = 0;
        for (int t = first_tile; t < tiles; t += tile_step) {
            const Tile w = tile_at<KIND>(table, p, t, group);
            const bool computed = w.blocks != 0;
            if (!computed && p.accumulate) continue;  // adds nothing
            const int acc = local & 1;
            if (computed) {
                const bool ok = ptx::mbar_wait(&bar.tmem_full[acc], (local >> 1) & 1, p.limit_ns, abort);
                if (!__all_sync(0xffffffffu, ok)) {
                    if (lane == 0) record_failure(p.status, abort, kRoleEpilogue);
                    break;
                }
                ++local;
                ptx::tc_fence_after();
            }
            const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                                   static_cast<uint32_t>(acc * kAccStep);
            const int n0 = w.n0 + rank * 128 + quarter * 32;
            if constexpr (!L::kGrad) {
#pragma unroll 1
                for (int c = 32 * turn; c < w.width; c += 64) {
                    uint32_t r[32];
                    load_rows_of_8(lanes + c, r);
                    store_transposed(r, staging, p.y + static_cast<int64_t>(w.b0 + c) * p.ldy, p.ldy, w.valid - c, n0, p.n,
                                     p.vec, lane);
                }
            } else {
                // Lanes are rows of the gradient: 32 rows of 128 bytes (64
                // columns, 32 in FP32) go through a swizzled buffer and out by
                // TMA, which clips them at the group's own edges: columns of a
                // last chunk past the width are past the row's end too.
                // (64-byte rows of BF16 took 311 us for 16 groups of 512 rows,
                // 4096 x 4096.)  A gradient that L2 cannot hold leaves it
                // first, in about the order it came (from 64 rows a group 112
                // us without, 91 with).
                const uint64_t policy = p.stream_out ? ptx::policy_evict_first() : ptx::policy_evict_normal();
                auto send = [&](int col) {
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0 && n0 < p.n && col < p.k) {
                        if (p.accumulate)
                            ptx::tma_add_3d(&map_c, staging, col, n0, p.first_group + w.e);
                        else
                            ptx::tma_store_3d_hint(&map_c, staging, col, n0, p.first_group + w.e, policy);
                        ptx::bulk_commit_group();
                    }
                };
                auto reusable = [&] {
                    if (lane == 0) ptx::bulk_wait_group_read<0>();
                    __syncwarp();
                };
#pragma unroll 1
                for (int c = 64 * turn; c < w.width; c += 128) {
                    uint32_t lo[32], hi[32];
                    if (computed) {
                        ptx::tmem_ld_32x32b_x32(lanes + c, lo);
                        ptx::tmem_ld_32x32b_x32(lanes + c + 32, hi);
                        ptx::tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) lo[j] = hi[j] = 0;
                    }
                    uint8_t* row = staging + lane * 128;
                    reusable();
                    if (p.fp32) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<uint4*>(row + (j ^ (lane & 7)) * 16) =
                                make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
                        send(w.b0 + c);
                        reusable();
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<uint4*>(row + (j ^ (lane & 7)) * 16) =
                                make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
                        send(w.b0 + c + 32);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t(&half)[32] = j < 4 ? lo : hi;
                            const int at = j % 4 * 8;
                            *reinterpret_cast<uint4*>(row + (j ^ (lane & 7)) * 16) =
                                make_uint4(gemm::pack_bf16x2(half[at], half[at + 1]),
                                           gemm::pack_bf16x2(half[at + 2], half[at + 3]),
                                           gemm::pack_bf16x2(half[at + 4], half[at + 5]),
                                           gemm::pack_bf16x2(half[at + 6], half[at + 7]));
                        }
                        send(w.b0 + c);
                    }
                }
            }
            if (computed) {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(ptx::smem_addr(&bar.tmem_empty[acc]), 0));
            }
        }
        if constexpr (L::kGrad) {
            if (lane == 0) ptx::bulk_wait_group_read<0>();  // shared memory outlives the stores' reads of it
        }
        __syncwarp();
    } else if (L::kMx && warp == kExtraWarp + 4) {
        // ------------------------------------------------- scales into TMEM
        // Per stage two words of 4 columns for the weight rows, two of 8 for
        // the tokens.  Its own thread issues the copies and a commit tells the
        // MMA's: issued by the MMA's thread itself they ran between its MMAs,
        // 50 cycles each (8192 x 8192 x 8192: 360 us, 277 apart).
        if (lane == 0 && leader) {
            Ring<S> ring;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += tile_step) {
                const Tile w = tile_at<KIND>(table, p, t, group);
                for (int kb = 0; kb < w.blocks; ++kb) {
                    if (!ptx::mbar_wait_cluster(&bar.full[ring.stage], ring.phase, p.limit_ns, abort)) {
                        record_failure(p.status, abort, kRoleMma);
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t ss =
                        ptx::smem_addr(smem + ring.stage * L::kStageBytes) + L::kABytes + L::kBBytes;
                    const uint32_t ts = tmem_base + 2 * kAccStep + ring.stage * L::kScaleCols;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        ptx::tmem_copy_scales<2>(ts + 4 * g, ptx::make_scale_desc(ss + 512 * g));
                        ptx::tmem_copy_scales<2>(ts + 8 + 8 * g, ptx::make_scale_desc(ss + 1024 + 1024 * g));
                        ptx::tmem_copy_scales<2>(ts + 12 + 8 * g, ptx::make_scale_desc(ss + 1536 + 1024 * g));
                    }
                    ptx::umma_commit_pair(&bar.copied[ring.stage], 1);
                    ring.next();
                }
            }
            // No copy is under way when the CTAs leave, whatever the MMAs did.
            ptx::umma_commit_pair(bar.copies_done, 1);
            if (!ptx::mbar_wait(bar.copies_done, 0, drain_limit(p.limit_ns), no_abort))
                record_failure(p.status, abort, kRoleDrain);
        }
        __syncwarp();
    } else if constexpr (L::kMx) {
        // -------------------------------------------------------------- scales
        // Thread i holds one of this CTA's 128 weight rows and two of the
        // tile's tokens (both CTAs need every token's scales): rows l / 4 + 32
        // (l % 4) + 8 warps for lane l, so that a warp's words lie side by side
        // in shared memory.  Scales come four stages at a time, two or three
        // 16-byte loads a row, and the next four stages' are under way while
        // these are handed out.
        const int i = (warp - kExtraWarp) * 8 + lane / 4 + lane % 4 * 32;
        const int blocks32 = p.k / 32;
        Ring<S> ring;
        bool ok = true;
        int t = first_tile, kb0 = 0;
        Tile w = {};
        const uint8_t* rows[3] = {};
        auto start_tile = [&] {
            w = tile_at<KIND>(table, p, t, group);
            const int n = w.n0 + rank * 128 + i;
            rows[0] = n < p.n ? p.w_scales + w.e * p.ws_stride + n * p.ldws : nullptr;
            for (int j = 0; j < 2; ++j)
                rows[1 + j] = i + 128 * j < w.valid ? p.x_scales + (static_cast<int64_t>(w.b0) + i + 128 * j) * p.ldxs : nullptr;
        };
        uint4 words[3][3], v[3][2];  // of each row: 32 scales for stages kb0 .. kb0 + 3, and the last four's
        auto load = [&] {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                load_scale_words(rows[j], kb0 * 8, blocks32, j == 0 ? p.w_span : p.x_span, words[j]);
        };
        if (t < tiles) {
            start_tile();
            load();
        }
        while (t < tiles && ok) {
#pragma unroll
            for (int j = 0; j < 3; ++j) align_scales(rows[j], kb0 * 8, blocks32, words[j], v[j]);
            const int here = min(4, w.blocks - kb0);
            kb0 += 4;
            if (kb0 >= w.blocks) {
                kb0 = 0;
                t += tile_step;
                if (t < tiles) start_tile();
            }
            if (t < tiles) load();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q >= here || !ok) break;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bar.empty[ring.stage], ring.phase ^ 1u, p.limit_ns, abort));
                if (!ok) {
                    if (lane == 0) record_failure(p.status, abort, kRoleProducer);
                    break;
                }
                uint8_t* ss = smem + ring.stage * L::kStageBytes + L::kABytes + L::kBBytes;
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    const uint4 both = v[j][q / 2];
                    const uint32_t at = j == 0 ? scale_word_offset(i) : 1024 + scale_word_offset(i + 128 * (j - 1));
                    *reinterpret_cast<uint32_t*>(ss + at) = q % 2 ? both.z : both.x;
                    *reinterpret_cast<uint32_t*>(ss + at + (j == 0 ? 512 : 1024)) = q % 2 ? both.w : both.y;
                }
                // The words are read by this CTA's own tensor core (through the
                // async proxy, which the fence orders them for), so the
                // arrival needs no release at cluster scope: that waits for
                // the loads under way as well, and made a stage 1.2 us long
                // (8192 x 8192 x 8192: 701 us).
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(ptx::smem_addr(&bar.full[ring.stage]), 0));
                ring.next();
            }
        }
        __syncwarp();
    } else if constexpr (L::kGrad) {
        // ---------------------------------------------------------------- tails
        Ring<S> ring;
        uint32_t landed_phase = 0;  // a bit per stage
        for (int t = first_tile; t < tiles; t += tile_step) {
            const Tile w = tile_at<KIND>(table, p, t, group);
            for (int kb = 0; kb < w.blocks - 1; ++kb) ring.next();
            if (w.blocks == 0) continue;
            if (w.tail != 0) {
                // Not cut short by a failure elsewhere: no copy may be in
                // flight when this CTA leaves.
                const bool ok = ptx::mbar_wait(&bar.landed[ring.stage], (landed_phase >> ring.stage) & 1u,
                                               drain_limit(p.limit_ns), no_abort);
                if (!__all_sync(0xffffffffu, ok)) {
                    if (lane == 0) record_failure(p.status, abort, kRoleProducer);
                    break;
                }
                landed_phase ^= 1u << ring.stage;
                // Rows tail .. next multiple of 16 of every box of their block:
                // 128 bytes each whatever the swizzle, which permutes within a
                // row.  (A multiple of 16 needs none.)
                const int block = w.tail / 64, first = w.tail % 64, count = round_up(w.tail, 16) - w.tail;
                uint8_t* stage = smem + ring.stage * L::kStageBytes;
                const int boxes = 2 + (w.width / 2 + 63) / 64;
                for (int i = lane; i < boxes * count * 8; i += 32) {
                    const int box = i / (count * 8), at = i % (count * 8);
                    uint8_t* base = box < 2 ? stage + block * L::kABlock + box * 8192
                                            : stage + L::kABytes + block * L::kBBlock + (box - 2) * 8192;
                    *reinterpret_cast<uint4*>(base + first * 128 + at * 16) = make_uint4(0, 0, 0, 0);
                }
                // Read by this CTA's own tensor core: see the scales' arrivals.
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(ptx::smem_addr(&bar.fixed[ring.stage]), 0));
            }
            ring.next();
        }
        __syncwarp();
    }

    if constexpr (!L::kGrad) {
        if (p.zero_rest) zero_rest_rows(p.y, p.ldy, table.rows(), p.rows, p.n, blockIdx.x, gridDim.x);
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        // Every UMMA that touches this CTA's memory has completed (the
        // leader's last commit arrives in both CTAs).
        if (lane == 0 && !ptx::mbar_wait(bar.drain, 0, drain_limit(p.limit_ns), no_abort))
            record_failure(p.status, abort, kRoleDrain);
        __syncwarp();
    }
    ptx::cluster_sync();  // no CTA leaves while its peer may still signal it
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

constexpr int kMaxDevices = 64;

template <Kind KIND>
int launch(const CUtensorMap& a, const CUtensorMap (&b)[3], const CUtensorMap& c, const PairParams& p, int64_t tiles,
           cudaStream_t stream) {
    using L = Pair<KIND>;
    static std::mutex mu;
    static bool configured[kMaxDevices] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return KMCTS_EHANDLE;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!configured[device]) {
            if (cudaFuncSetAttribute(grouped_pair_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     L::smem_bytes(L::kMaxGroups)) != cudaSuccess)
                return KMCTS_EGEMM;
            configured[device] = true;
        }
    }
    const int64_t pairs = multiprocessor_count() / 2;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    allow_early_start(&attr[1]);
    config.gridDim = dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)), 1, 1);
    config.blockDim = dim3(L::kThreads, 1, 1);
    config.dynamicSmemBytes = L::smem_bytes(p.groups);
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = 2;
    const cudaError_t err = cudaLaunchKernelEx(&config, grouped_pair_kernel<KIND>, a, b[0], b[1], b[2], c, p);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (err == cudaSuccess) return KMCTS_OK;
    cudaGetLastError();  // reported here, not by the caller's next call
    return KMCTS_EGEMM;
}

}  // namespace

int launch_forward_pair(const ForwardArgs& f, Operand operand, uint64_t limit_ns, cudaStream_t stream, int* status) {
    PairParams p = {};
    p.ends = f.ends, p.groups = f.groups, p.rows = f.rows, p.n = f.n, p.k = f.k;
    p.y = static_cast<__nv_bfloat16*>(f.y), p.ldy = f.ldy;
    p.vec = reinterpret_cast<uintptr_t>(f.y) % 16 == 0 && f.ldy % 8 == 0;
    p.zero_rest = f.zero_rest;
    p.x_scales = f.x_scales, p.ldxs = f.ldxs;
    p.w_scales = f.w_scales, p.ws_stride = f.ws_stride, p.ldws = f.ldws;
    scale_spans(f, &p.x_span, &p.w_span);
    p.limit_ns = limit_ns, p.status = status;
    const bool mx = operand == Operand::kMxfp4;
    const uint32_t box_rows[3] = {mx ? 96u : 128u, 64, 32};
    CUtensorMap a, b[3];
    if (!encode_forward_maps(f, operand, &a, b, box_rows)) return KMCTS_ENOTSUP;
    p.strip = Divisor::of(8 * ((f.n + 255) / 256));
    const int64_t width = mx ? 192 : 256;
    const int64_t tiles = (f.rows / width + f.groups) * ((f.n + 255) / 256);
    if (tiles >= 1LL << 30) return KMCTS_ENOTSUP;
    switch (operand) {
        case Operand::kBf16Col: return launch<Kind::kCol>(a, b, a, p, tiles, stream);
        case Operand::kBf16Row: return launch<Kind::kRow>(a, b, a, p, tiles, stream);
        case Operand::kMxfp4: return launch<Kind::kMxfp4>(a, b, a, p, tiles, stream);
    }
    return KMCTS_EINVAL;
}

int launch_wgrad_pair(const WgradArgs& g, uint64_t limit_ns, cudaStream_t stream, int* status) {
    const int64_t tiles = static_cast<int64_t>(g.groups) * ((g.n + 255) / 256) * ((g.k + 255) / 256);
    if (tiles >= 1LL << 30) return KMCTS_ENOTSUP;
    PairParams p = {};
    p.ends = g.ends, p.groups = g.groups, p.rows = g.rows, p.n = g.n, p.k = g.k;
    p.fp32 = g.fp32, p.accumulate = g.accumulate;
    p.limit_ns = limit_ns, p.status = status;
    const uint64_t n = g.n, k = g.k, rows = g.rows;
    CUtensorMap a, b[3], c;
    auto encode_rows = [&](CUtensorMap* map, const void* base, uint64_t cols, int64_t ld) {
        const uint64_t dims[2] = {cols, rows}, strides[1] = {static_cast<uint64_t>(ld) * 2};
        const uint32_t box[2] = {64, 64};
        return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (!encode_rows(&a, g.dy, n, g.lddy) || !encode_rows(&b[1], g.x, k, g.ldx)) return KMCTS_ENOTSUP;
    b[0] = b[2] = b[1];  // not used
    {
        const uint64_t size = g.fp32 ? 4 : 2;
        const uint64_t group = g.groups > 1 ? g.dw_stride : g.lddw * n;
        const uint64_t dims[3] = {k, n, static_cast<uint64_t>(g.groups)}, strides[2] = {g.lddw * size, group * size};
        const uint32_t box[3] = {g.fp32 ? 32u : 64u, 32, 1};
        if (!encode_map(&c, g.fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, g.dw, dims,
                        strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
            return KMCTS_ENOTSUP;
    }
    p.strip = Divisor::of(8 * ((g.k + 255) / 256));
    p.per_group = Divisor::of(static_cast<uint32_t>(tiles / g.groups));
    p.stream_out = static_cast<int64_t>(g.groups) * g.n * g.k * (g.fp32 ? 4 : 2) > 63LL << 20;  // L2 is 126 MB
    constexpr int most = Pair<Kind::kWgrad>::kMaxGroups;
    for (; p.first_group < g.groups; p.first_group += most) {
        p.groups = g.groups - p.first_group < most ? g.groups - p.first_group : most;
        const int rc = launch<Kind::kWgrad>(a, b, c, p, static_cast<int64_t>(p.groups) * p.per_group.d, stream);
        if (rc != KMCTS_OK) return rc;
    }
    return KMCTS_OK;
}

}  // namespace grouped
}  // namespace kmcts
