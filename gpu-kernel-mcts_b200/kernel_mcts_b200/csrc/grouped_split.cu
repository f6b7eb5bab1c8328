// Grouped products for few rows a group (decoding): bound by reading the
// weights, so what counts is that every SM streams them all the time.
//
// As in grouped_pair.cu the weight is the MMA's A and the tokens its N, here
// 128 weight rows x up to 64 tokens on one CTA, so the MMA's work follows the
// token count in steps of 16.  A cluster of S CTAs shares a tile: each takes a
// contiguous part of K, so that few tiles still keep every SM busy and no
// workspace is needed.  The CTAs' FP32 parts meet in shared memory: quarter q
// of the tile's rows belongs to CTA q % S, every CTA stores its part of the
// quarter there (asynchronous stores, counted in bytes), and the owner adds
// the S parts in K order, rounds once and writes 64-byte pieces of token rows.
// The order of the sum is fixed, so repeated calls give the same bits.
//
// Roles per CTA as in grouped_pair.cu: producer, MMA, four epilogue warps; for
// MXFP4 four warps that fetch scales and one that issues their copies.
#include <mutex>

#include "grouped_tiles.cuh"

namespace kmcts {
namespace grouped {
namespace {

constexpr int kBaseThreads = 192;
constexpr int kMaxWidth = 64;  // tokens of a tile
constexpr int kMaxSplits = 4;
constexpr int kPartBytes = 32 * kMaxWidth * 4;  // one CTA's part of one quarter

template <Kind KIND>
struct Split {
    static constexpr bool kMx = KIND == Kind::kMxfp4;
    static constexpr bool kAMn = KIND == Kind::kRow;
    static constexpr int kThreads = kBaseThreads + (kMx ? 160 : 0);
    static constexpr int kBK = kMx ? 256 : 64;
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = kMaxWidth * 128;
    static constexpr int kScaleBytes = kMx ? 2 * 512 + 2 * 512 : 0;
    static constexpr int kStageBytes = kABytes + kBBytes + kScaleBytes;
    static constexpr int kStages = 7;
    static constexpr int kScaleCols = 16;  // a stage's: 2 x 4 for the weight rows, 2 x 4 for the tokens
    static constexpr int kTmemCols = kMx ? 256 : 128;
    // Each CTA owns 4 / S quarters, S parts of each: four parts whatever S is.
    static constexpr int kPartsOffset = kStages * kStageBytes;
    static constexpr int kBarrierOffset = kPartsOffset + 4 * kPartBytes;
    static constexpr int kTableOffset = kBarrierOffset + 512;
    static constexpr int smem_bytes(int groups) { return 1024 + kTableOffset + table_bytes(groups, false); }
    static_assert(2 * kMaxWidth + (kMx ? kStages * kScaleCols : 0) <= kTmemCols, "TMEM columns");
    static_assert(smem_bytes(KMCTS_MAX_GROUPS) <= kMaxSmem, "shared memory");
};

struct SplitParams {
    const int32_t* ends;
    int groups, rows, n, k;
    __nv_bfloat16* y;
    int64_t ldy;
    bool zero_rest;
    const uint8_t* x_scales;
    int64_t ldxs;
    const uint8_t* w_scales;
    int64_t ws_stride, ldws;
    ScaleSpan x_span, w_span;
    uint64_t limit_ns;
    int* status;
};

// Weight rows from n0, tokens from t0 (`width` computed, `valid` stored), and
// this CTA's stages [kb0, kb1) of K.
struct Tile {
    int e, n0, t0, width, valid, kb0, kb1;
};

template <Kind KIND>
__device__ __forceinline__ Tile tile_at(const GroupTable& table, const SplitParams& p, int t, int rank, int splits,
                                        int& group) {
    Tile out;
    out.e = group_of_tile(table, t, group);
    const int in_group = t - table.tile[out.e];
    const int first = table.row[out.e], rows = table.row[out.e + 1] - first;
    const int tiles_t = (rows + kMaxWidth - 1) / kMaxWidth;
    const int step = tiles_t == 1 ? round_up(rows, 16) : round_up((rows + tiles_t - 1) / tiles_t, 16);
    // A weight tile's token tiles follow one another: its second reading is
    // from L2.
    const int n_blk = tiles_t == 1 ? in_group : in_group / tiles_t;
    out.n0 = n_blk * 128;
    out.t0 = first + (in_group - n_blk * tiles_t) * step;
    out.valid = min(step, first + rows - out.t0);
    out.width = round_up(out.valid, 16);
    // Splits are 2 or 4.
    const int blocks = (p.k + Split<KIND>::kBK - 1) / Split<KIND>::kBK, shift = splits >> 1;
    out.kb0 = static_cast<int>(static_cast<int64_t>(rank) * blocks >> shift);
    out.kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * blocks >> shift);
    return out;
}

template <Kind KIND>
__global__ void __launch_bounds__(Split<KIND>::kThreads, 1)
    grouped_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b64,
                         const __grid_constant__ CUtensorMap map_b32, const __grid_constant__ CUtensorMap map_b16,
                         const __grid_constant__ SplitParams p) {
    using L = Split<KIND>;
    constexpr int S = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarrierOffset);
    uint64_t* empty = full + S;
    uint64_t* copied = empty + S;
    uint64_t* tmem_full = copied + S;
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* drain = tmem_empty + 2;
    uint64_t* copies_done = drain + 1;
    uint64_t* arrived = copies_done + 1;  // every part of this CTA's quarters is here
    uint64_t* freed = arrived + 1;        // quarter q's owner has read the last tile's parts
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(freed + 4);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* no_abort = abort + 1;
    int* table_smem = reinterpret_cast<int*>(smem + L::kTableOffset);
    const GroupTable table(table_smem, p.groups);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = static_cast<int>(ptx::cluster_ctarank());
    const int splits = static_cast<int>(ptx::cluster_nctarank());
    const int first_tile = blockIdx.x / splits, tile_step = gridDim.x / splits;

    ptx::let_next_grid_start();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            ptx::mbar_init(&full[s], L::kMx ? 5 : 1);  // MXFP4: the byte count and four scale warps
            ptx::mbar_init(&empty[s], 1);
            ptx::mbar_init(&copied[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(&tmem_full[a], 1);
            ptx::mbar_init(&tmem_empty[a], 4);
        }
        ptx::mbar_init(drain, 1);
        ptx::mbar_init(copies_done, 1);
        ptx::mbar_init(arrived, 1);
        for (int q = 0; q < 4; ++q) ptx::mbar_init(&freed[q], 4);
        *abort = 0;
        *no_abort = 0;
        ptx::fence_mbarrier_init();
        ptx::prefetch_tensormap(&map_a);
        ptx::prefetch_tensormap(&map_b64);
        ptx::prefetch_tensormap(&map_b32);
        ptx::prefetch_tensormap(&map_b16);
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, L::kTmemCols);
        ptx::tmem_relinquish();
    }
    // Up to here the launch overlaps the end of the grid before.
    ptx::wait_for_earlier_grids();
    if (warp == 2) {
        const int tiles_n = (p.n + 127) / 128;
        build_group_table(table, p.ends, p.rows,
                          [&](int rows) { return (rows + kMaxWidth - 1) / kMaxWidth * tiles_n; });
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int tiles = table.tiles();
    int group = 0;  // the last tile's

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            // The weights are read once: they leave L2 first.
            const uint64_t once = ptx::policy_evict_first();
            Ring<S> ring;
            uint32_t issued = 0, issued_phase = 0;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += tile_step) {
                const Tile w = tile_at<KIND>(table, p, t, rank, splits, group);
                const CUtensorMap* mb = w.width > 32 ? &map_b64 : w.width > 16 ? &map_b32 : &map_b16;
                const int box_rows = w.width > 32 ? 64 : w.width > 16 ? 32 : 16;
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    if (!ptx::mbar_wait(&empty[ring.stage], ring.phase ^ 1u, p.limit_ns, abort)) {
                        record_failure(p.status, abort, kRoleProducer);
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + ring.stage * L::kStageBytes;
                    uint64_t* bar = &full[ring.stage];
                    ptx::mbar_arrive_expect_tx(bar, static_cast<uint32_t>(L::kABytes + box_rows * 128));
                    const int k0 = kb * (L::kMx ? 128 : 64);  // MXFP4 maps count bytes
                    if constexpr (L::kAMn) {
                        for (int i = 0; i < 2; ++i)
                            ptx::tma_load_3d_hint(sa + i * 8192, &map_a, bar, w.n0 + 64 * i, k0, w.e, once);
                    } else {
                        ptx::tma_load_3d_hint(sa, &map_a, bar, k0, w.n0, w.e, once);
                    }
                    ptx::tma_load_2d(sa + L::kABytes, mb, bar, k0, w.t0);
                    issued |= 1u << ring.stage;
                    issued_phase = (issued_phase & ~(1u << ring.stage)) | (ring.phase << ring.stage);
                    ring.next();
                }
            }
            for (int s = 0; s < S; ++s) {  // no copy is under way when this CTA leaves
                if ((issued & (1u << s)) &&
                    !ptx::mbar_wait(&full[s], (issued_phase >> s) & 1u, drain_limit(p.limit_ns), no_abort))
                    record_failure(p.status, abort, kRoleDrain);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ----------------------------------------------------------------- MMA
        if (lane == 0) {
            Ring<S> ring;
            int local = 0;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += tile_step) {
                const Tile w = tile_at<KIND>(table, p, t, rank, splits, group);
                if (w.kb0 == w.kb1) continue;
                const int acc = local & 1;
                if (!ptx::mbar_wait(&tmem_empty[acc], ((local >> 1) & 1) ^ 1u, p.limit_ns, abort)) {
                    record_failure(p.status, abort, kRoleMma);
                    break;
                }
                ++local;
                ptx::tc_fence_after();
                const uint32_t d = tmem_base + acc * kMaxWidth;
                const uint32_t idesc = L::kMx ? ptx::make_idesc_mxf4(128, w.width, 0)
                                              : ptx::make_idesc_bf16_ab(128, w.width, L::kAMn, false);
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    if (!ptx::mbar_wait(L::kMx ? &copied[ring.stage] : &full[ring.stage], ring.phase, p.limit_ns, abort)) {
                        record_failure(p.status, abort, kRoleMma);
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t sa = ptx::smem_addr(smem + ring.stage * L::kStageBytes);
                    const uint32_t sb = sa + L::kABytes;
                    const uint32_t ts = tmem_base + 2 * kMaxWidth + ring.stage * L::kScaleCols;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const bool add = kb != w.kb0 || kk != 0;
                        const uint64_t bdesc = ptx::make_sw128_desc(sb + kk * 32, 16, 1024);
                        if constexpr (L::kMx) {
                            const uint32_t id = static_cast<uint32_t>(kk % 2 * 2);
                            ptx::umma_mxf4<1>(d, ptx::make_sw128_desc(sa + kk * 32, 16, 1024), bdesc,
                                              idesc | id << 4 | id << 29, ts + 4 * (kk / 2), ts + 8 + 4 * (kk / 2), add);
                        } else {
                            ptx::umma_bf16(d,
                                           L::kAMn ? ptx::make_sw128_desc(sa + kk * 2048, 8192, 1024)
                                                   : ptx::make_sw128_desc(sa + kk * 32, 16, 1024),
                                           bdesc, idesc, add);
                        }
                    }
                    ptx::umma_commit(&empty[ring.stage]);
                    ring.next();
                }
                if (ok) ptx::umma_commit(&tmem_full[acc]);
            }
            ptx::umma_commit(drain);
        }
        __syncwarp();
    } else if (warp < 6) {
        // ------------------------------------------------------------ epilogue
        const int quarter = warp % 4;
        const int owner = quarter % splits;
        float* parts = reinterpret_cast<float*>(smem + L::kPartsOffset);
        // This CTA's part of its quarter, in the owner's shared memory: slot
        // (quarter / S) * S + rank.
        const uint32_t mine = ptx::mapa_shared(
            ptx::smem_addr(parts) + (quarter / splits * splits + rank) * kPartBytes + lane * 16, owner);
        const uint32_t mine_arrived = ptx::mapa_shared(ptx::smem_addr(arrived), owner);
        int local = 0, seen = 0;
        bool ok = true;
        for (int t = first_tile; t < tiles && ok; t += tile_step, ++seen) {
            const Tile w = tile_at<KIND>(table, p, t, rank, splits, group);
            const bool computed = w.kb0 != w.kb1;
            const int acc = local & 1;
            if (computed) {
                ok = ptx::mbar_wait(&tmem_full[acc], (local >> 1) & 1, p.limit_ns, abort);
                ++local;
            }
            if (ok && seen > 0) ok = ptx::mbar_wait_cluster(&freed[quarter], (seen - 1) & 1, p.limit_ns, abort);
            // Four parts of width x 32 values come here, whatever S is.  Their
            // stores are asynchronous: a CTA that gives up still waits
            // (bounded) for the other CTAs' before it leaves.
            const uint32_t part_bytes = static_cast<uint32_t>(w.width * 512);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0) record_failure(p.status, abort, kRoleEpilogue);
                if (threadIdx.x == 64) ptx::mbar_arrive_expect_tx(arrived, part_bytes);
                ptx::mbar_wait_cluster(arrived, seen & 1, drain_limit(p.limit_ns), no_abort);
                break;
            }
            ptx::tc_fence_after();
            const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                                   static_cast<uint32_t>(acc * kMaxWidth);
            // Four tokens' values of a row at a time: [token / 4][row][token % 4].
#pragma unroll 1
            for (int c = 0; c < w.width; c += 32) {
                uint32_t r[32];
                if (computed) {
                    ptx::tmem_ld_32x32b_x32(lanes + c, r);
                    ptx::tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0;
                }
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    if (c + 4 * g < w.width)
                        ptx::st_async_v4(mine + (c / 4 + g) * 512, r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3],
                                         mine_arrived);
            }
            if (computed) {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&tmem_empty[acc]);
            }
            if (threadIdx.x == 64) ptx::mbar_arrive_expect_tx(arrived, part_bytes);
            // The parts of this CTA's quarters: the four warps share the tokens.
            ok = __all_sync(0xffffffffu, ptx::mbar_wait_cluster(arrived, seen & 1, drain_limit(p.limit_ns), no_abort));
            if (!ok) {
                if (lane == 0) record_failure(p.status, abort, kRoleEpilogue);
                break;
            }
            for (int q = rank; q < 4; q += splits) {
                const float4* part = reinterpret_cast<const float4*>(parts) + q / splits * splits * (kPartBytes / 16) + lane;
                const int col = w.n0 + q * 32 + lane;
                for (int g = warp - 2; g < w.width / 4; g += 4) {
                    float4 sum = part[g * 32];
                    for (int s = 1; s < splits; ++s) {
                        const float4 v = part[s * (kPartBytes / 16) + g * 32];
                        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                    }
                    const float values[4] = {sum.x, sum.y, sum.z, sum.w};
                    __nv_bfloat16* dst = p.y + (static_cast<int64_t>(w.t0) + 4 * g) * p.ldy + col;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col < p.n && 4 * g + j < w.valid) dst[j * p.ldy] = __float2bfloat16_rn(values[j]);
                }
                // The parts have been read (their sums are stored), which is
                // all that the next ones wait for: no release of the stores
                // to Y, which would wait for memory.
                __syncwarp();
                if (lane < splits) ptx::mbar_arrive_cluster(ptx::mapa_shared(ptx::smem_addr(&freed[q]), lane));
            }
        }
        __syncwarp();
    } else if (L::kMx && warp == 10) {
        // ------------------------------------------------- scales into TMEM
        if (lane == 0) {
            Ring<S> ring;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += tile_step) {
                const Tile w = tile_at<KIND>(table, p, t, rank, splits, group);
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    if (!ptx::mbar_wait(&full[ring.stage], ring.phase, p.limit_ns, abort)) {
                        record_failure(p.status, abort, kRoleMma);
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t ss = ptx::smem_addr(smem + ring.stage * L::kStageBytes) + L::kABytes + L::kBBytes;
                    const uint32_t ts = tmem_base + 2 * kMaxWidth + ring.stage * L::kScaleCols;
#pragma unroll
                    for (int g = 0; g < 4; ++g) ptx::tmem_copy_scales<1>(ts + 4 * g, ptx::make_scale_desc(ss + 512 * g));
                    ptx::umma_commit(&copied[ring.stage]);
                    ring.next();
                }
            }
            ptx::umma_commit(copies_done);
            if (!ptx::mbar_wait(copies_done, 0, drain_limit(p.limit_ns), no_abort))
                record_failure(p.status, abort, kRoleDrain);
        }
        __syncwarp();
    } else if constexpr (L::kMx) {
        // -------------------------------------------------------------- scales
        // As in grouped_pair.cu; thread i holds weight row i and token i.
        const int i = (warp - 6) * 8 + lane / 4 + lane % 4 * 32;
        const int blocks32 = p.k / 32;
        Ring<S> ring;
        bool ok = true;
        int t = first_tile, kb = 0;
        Tile w = {};
        const uint8_t* rows[2] = {};
        // Groups of four stages start at multiples of four, whatever this
        // CTA's first stage is: loads are aligned.
        auto start_tile = [&] {
            for (; t < tiles; t += tile_step) {
                w = tile_at<KIND>(table, p, t, rank, splits, group);
                if (w.kb0 < w.kb1) break;
            }
            if (t >= tiles) return;
            kb = w.kb0;
            const int n = w.n0 + i;
            rows[0] = n < p.n ? p.w_scales + w.e * p.ws_stride + n * p.ldws : nullptr;
            rows[1] = i < w.valid ? p.x_scales + (static_cast<int64_t>(w.t0) + i) * p.ldxs : nullptr;
        };
        uint4 words[2][3], v[2][2];
        auto load = [&] {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                load_scale_words(rows[j], kb / 4 * 32, blocks32, j == 0 ? p.w_span : p.x_span, words[j]);
        };
        start_tile();
        if (t < tiles) load();
        while (t < tiles && ok) {
#pragma unroll
            for (int j = 0; j < 2; ++j) align_scales(rows[j], kb / 4 * 32, blocks32, words[j], v[j]);
            const int from = kb % 4, to = min(4, w.kb1 - kb / 4 * 4);
            kb = (kb / 4 + 1) * 4;
            if (kb >= w.kb1) {
                t += tile_step;
                start_tile();
            }
            if (t < tiles) load();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q < from || q >= to || !ok) continue;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&empty[ring.stage], ring.phase ^ 1u, p.limit_ns, abort));
                if (!ok) {
                    if (lane == 0) record_failure(p.status, abort, kRoleProducer);
                    continue;
                }
                uint8_t* ss = smem + ring.stage * L::kStageBytes + L::kABytes + L::kBBytes + scale_word_offset(i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 both = v[j][q / 2];
                    *reinterpret_cast<uint32_t*>(ss + 1024 * j) = q % 2 ? both.z : both.x;
                    *reinterpret_cast<uint32_t*>(ss + 1024 * j + 512) = q % 2 ? both.w : both.y;
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&full[ring.stage]);
                ring.next();
            }
        }
        __syncwarp();
    }

    if (p.zero_rest) zero_rest_rows(p.y, p.ldy, table.rows(), p.rows, p.n, blockIdx.x, gridDim.x);
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (lane == 0 && !ptx::mbar_wait(drain, 0, drain_limit(p.limit_ns), no_abort))
            record_failure(p.status, abort, kRoleDrain);
        __syncwarp();
    }
    ptx::cluster_sync();  // no CTA leaves while another may still write its parts
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, L::kTmemCols);
    }
}

constexpr int kMaxDevices = 64;

// Clusters of `splits` CTAs that are resident at once, from the occupancy
// calculator (GPCs hold whole clusters only, so this is less than SMs / splits
// for four); the kernel's shared-memory limit is raised on the way.
template <Kind KIND>
int resident_clusters(int device, int splits) {
    using L = Split<KIND>;
    static std::mutex mu;
    static int known[kMaxDevices][kMaxSplits + 1] = {};
    std::lock_guard<std::mutex> lock(mu);
    int& clusters = known[device][splits];
    if (clusters > 0) return clusters;
    if (cudaFuncSetAttribute(grouped_split_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             L::smem_bytes(KMCTS_MAX_GROUPS)) != cudaSuccess)
        return -1;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.gridDim = dim3(splits * (multiprocessor_count() / splits), 1, 1);
    config.blockDim = dim3(L::kThreads, 1, 1);
    config.dynamicSmemBytes = L::smem_bytes(KMCTS_MAX_GROUPS);
    config.attrs = attr;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters, grouped_split_kernel<KIND>, &config) != cudaSuccess || clusters <= 0) {
        cudaGetLastError();
        clusters = multiprocessor_count() / splits;
    }
    return clusters;
}

template <Kind KIND>
int launch(const CUtensorMap& a, const CUtensorMap (&b)[3], const SplitParams& p, int64_t tiles, int splits,
           cudaStream_t stream) {
    using L = Split<KIND>;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return KMCTS_EHANDLE;
    const int64_t clusters = resident_clusters<KIND>(device, splits);
    if (clusters <= 0) return KMCTS_EGEMM;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    allow_early_start(&attr[1]);
    config.gridDim = dim3(static_cast<unsigned>(splits * (tiles < clusters ? tiles : clusters)), 1, 1);
    config.blockDim = dim3(L::kThreads, 1, 1);
    config.dynamicSmemBytes = L::smem_bytes(p.groups);
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = 2;
    const cudaError_t err = cudaLaunchKernelEx(&config, grouped_split_kernel<KIND>, a, b[0], b[1], b[2], p);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (err == cudaSuccess) return KMCTS_OK;
    cudaGetLastError();  // reported here, not by the caller's next call
    return KMCTS_EGEMM;
}

}  // namespace

int launch_forward_split(const ForwardArgs& f, Operand operand, int splits, uint64_t limit_ns, cudaStream_t stream,
                         int* status) {
    SplitParams p = {};
    p.ends = f.ends, p.groups = f.groups, p.rows = f.rows, p.n = f.n, p.k = f.k;
    p.y = static_cast<__nv_bfloat16*>(f.y), p.ldy = f.ldy;
    p.zero_rest = f.zero_rest;
    p.x_scales = f.x_scales, p.ldxs = f.ldxs;
    p.w_scales = f.w_scales, p.ws_stride = f.ws_stride, p.ldws = f.ldws;
    scale_spans(f, &p.x_span, &p.w_span);
    p.limit_ns = limit_ns, p.status = status;
    static const uint32_t box_rows[3] = {64, 32, 16};
    CUtensorMap a, b[3];
    if (!encode_forward_maps(f, operand, &a, b, box_rows)) return KMCTS_ENOTSUP;
    const int64_t tiles = (f.rows / kMaxWidth + (f.groups < f.rows ? f.groups : f.rows)) *
                          static_cast<int64_t>((f.n + 127) / 128);
    if (tiles >= 1LL << 30) return KMCTS_ENOTSUP;
    switch (operand) {
        case Operand::kBf16Col: return launch<Kind::kCol>(a, b, p, tiles, splits, stream);
        case Operand::kBf16Row: return launch<Kind::kRow>(a, b, p, tiles, splits, stream);
        case Operand::kMxfp4: return launch<Kind::kMxfp4>(a, b, p, tiles, splits, stream);
    }
    return KMCTS_EINVAL;
}

}  // namespace grouped
}  // namespace kmcts
