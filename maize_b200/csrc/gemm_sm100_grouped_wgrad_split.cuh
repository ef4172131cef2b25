// The weight gradient of the grouped product where the tiles are too few to fill the SMs (one or a few groups of many rows,
// small matrices): a cluster of S = 2, 4 or 8 CTAs shares a 128 x 128 tile of DW and splits the group's ROWS.
//
// Each CTA multiplies its blocks of 64 rows (both operands MN-major, rows past the group's end cleared by the fix warp, as in
// gemm_sm100_grouped_wgrad.cuh) into its own tensor memory.  The parts meet in distributed shared memory: every CTA finishes
// 128 / S columns of the tile, adds the S parts in the order of the rows, rounds once and stores.
//
// Bound: the latency of one CTA's blocks of rows, about 0.3 us each; 11186 rows, 136 x 544: 15 us instead of 61.
#pragma once
#include "gemm_sm100_grouped_wgrad.cuh"

namespace maize {

constexpr uint32_t kWgradSplitTile = 128;  // rows and columns of DW per tile
constexpr uint32_t kWgradSplitThreads = 224;

template <uint32_t S, uint32_t STAGES>
struct WgradSplitLayout {
    static constexpr uint32_t kShare = kWgradSplitTile / S;             // columns that one CTA finishes
    static constexpr uint32_t kOperandBytes = kBlockM * kBlockK * 2;    // two boxes of 64 columns x 64 rows
    static constexpr uint32_t kStageBytes = 2 * kOperandBytes;          // [DC0, DC1, A0, A1]
    static constexpr uint32_t kExchangeOffset = STAGES * kStageBytes;   // from each other CTA: [warp][4 columns][lane]
    static constexpr uint32_t kWarpBytes = kShare * 32 * 4;
    static constexpr uint32_t kPartBytes = kNumEpilogueWarps * kWarpBytes;
    static constexpr uint32_t kBarOffset = kExchangeOffset + (S - 1) * kPartBytes;
    static constexpr uint32_t kNumBars = 3 * STAGES + 4 + 2;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kTableOffset = (kAbortOffset + 4 + 15) / 16 * 16;
    static constexpr uint32_t kUsedBytes = kTableOffset + kGroupTableBytes;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
    static_assert(kWarpBytes >= 32 * kShare * 2, "a warp's part of the exchange serves as its staging buffer");
};

// One tile, and the blocks of 64 rows that CTA `rank` of the cluster multiplies.
struct WgradSplitTile {
    uint32_t group, m0, n0;       // first row and column of DW
    uint32_t row0, rows, blocks;  // first row of this CTA's part, rows and blocks in it
};

template <uint32_t S>
__device__ __forceinline__ WgradSplitTile wgrad_split_tile(uint32_t t, uint32_t m_blocks, uint32_t n_blocks, uint32_t rank,
                                                           const GroupTable &tab)
{
    const uint32_t per_group = m_blocks * n_blocks;
    WgradSplitTile r;
    const uint32_t at = t / per_group, local = t - at * per_group;
    r.group = tab.order[at];
    r.m0 = local / n_blocks * kWgradSplitTile;
    r.n0 = local % n_blocks * kWgradSplitTile;
    const uint32_t begin = tab.offset[r.group], all = tab.offset[r.group + 1] - begin;
    const uint32_t all_blocks = (all + kBlockK - 1) / kBlockK, per_cta = (all_blocks + S - 1) / S;
    const uint32_t first = min(rank * per_cta, all_blocks);
    r.blocks = min(per_cta, all_blocks - first);
    r.row0 = begin + first * kBlockK;
    r.rows = r.blocks == 0 ? 0u : min(r.blocks * kBlockK, all - first * kBlockK);
    return r;
}

template <uint32_t S, uint32_t STAGES>
__global__ void __launch_bounds__(kWgradSplitThreads, 1)
gemm_bf16_sm100_grouped_wgrad_split(const __grid_constant__ CUtensorMap tma_dc, const __grid_constant__ CUtensorMap tma_a,
                                    const GroupedParams p)
{
    using L = WgradSplitLayout<S, STAGES>;
    constexpr uint32_t kTmemCols = 2 * kWgradSplitTile;
    constexpr uint32_t kChunkBytes = kBlockK * 128;
    constexpr uint32_t kIdesc = ptx::make_instr_desc_bf16(kBlockM, kWgradSplitTile, true, true);

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto tail_bar = [&](uint32_t s) { return bar_base + 8u * (2 * STAGES + s); };  // the bytes of a cut block
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (3 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (3 * STAGES + 2 + b); };
    const uint32_t sums_full_bar = bar_base + 8u * (3 * STAGES + 4);   // the other CTAs' sums are here
    const uint32_t sums_taken_bar = bar_base + 8u * (3 * STAGES + 5);  // the others have read what this CTA sent
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);
    const GroupTable tab(smem_gen + L::kTableOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t rank = ptx::cluster_cta_rank();
    const uint32_t cluster = blockIdx.x / S;
    const uint32_t num_clusters = gridDim.x / S;
    const uint32_t m_blocks = (p.n + kWgradSplitTile - 1) / kWgradSplitTile;
    const uint32_t n_blocks = (p.k + kWgradSplitTile - 1) / kWgradSplitTile;
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_dc);
        ptx::prefetch_tensormap(&tma_a);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);  // the producer and the bytes, or the fix warp
            ptx::mbar_init(empty_bar(s), 1);
            ptx::mbar_init(tail_bar(s), 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            ptx::mbar_init(acc_full_bar(b), 1);
            ptx::mbar_init(acc_empty_bar(b), kNumEpilogueWarps);
        }
        ptx::mbar_init(sums_full_bar, (S - 1) * kNumEpilogueWarps);
        ptx::mbar_init(sums_taken_bar, (S - 1) * kNumEpilogueWarps);
        *abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc_1cta(ptx::smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemCols);
        ptx::tmem_relinquish_1cta();
    }
    ptx::tcgen05_fence_before();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    ptx::tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (p.pdl) {
        if (threadIdx.x == 0)
            ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t all_tiles = p.groups * m_blocks * n_blocks;
    const uint32_t num_tiles = build_wgrad_table(p, tab, all_tiles <= num_clusters) ? all_tiles : 0u;

    bool role_ok = true;
    if (warp == 0) {
        // ------------------------------------------------------- TMA producer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint64_t round = 0, t; ok && (t = dealt_tile(round, cluster, num_clusters)) < num_tiles; ++round) {
                const WgradSplitTile tile = wgrad_split_tile<S>(static_cast<uint32_t>(t), m_blocks, n_blocks, rank, tab);
                for (uint32_t b = 0; b < tile.blocks; ++b) {
                    ok = wait_bounded(empty_bar(stage), phase ^ 1u, ctl, 1);
                    if (!ok)
                        break;
                    const uint32_t sd = smem_base + stage * L::kStageBytes;
                    const uint32_t sa = sd + L::kOperandBytes;
                    const int32_t r = static_cast<int32_t>(tile.row0 + b * kBlockK);
                    const uint32_t left = tile.rows - b * kBlockK;
                    // the bytes of a cut block go by the fix warp
                    const uint32_t bar = left < kBlockK && (left & 15u) != 0u ? tail_bar(stage) : full_bar(stage);
                    ptx::mbar_arrive_expect_tx(bar, L::kStageBytes);
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j) {
                        ptx::tma_load_2d(sd + j * kChunkBytes, &tma_dc, bar, static_cast<int32_t>(tile.m0 + 64u * j), r);
                        ptx::tma_load_2d(sa + j * kChunkBytes, &tma_a, bar, static_cast<int32_t>(tile.n0 + 64u * j), r);
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            role_ok = ok;
        }
        __syncwarp();
    } else if (warp == 1) {
        // -------------------------------------------------------- MMA issuer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            uint32_t acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint64_t round = 0, t; ok && (t = dealt_tile(round, cluster, num_clusters)) < num_tiles; ++round) {
                const WgradSplitTile tile = wgrad_split_tile<S>(static_cast<uint32_t>(t), m_blocks, n_blocks, rank, tab);
                if (tile.blocks == 0)
                    continue;  // nothing of this tile here: no accumulator changes hands
                ok = wait_bounded(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t tmem_d = tmem_base + acc * kWgradSplitTile;
                for (uint32_t b = 0; b < tile.blocks; ++b) {
                    ok = wait_bounded(full_bar(stage), phase, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sd = smem_base + stage * L::kStageBytes;
                    const uint64_t dd = ptx::make_smem_desc_sw128_mn(sd, kChunkBytes);
                    const uint64_t da = ptx::make_smem_desc_sw128_mn(sd + L::kOperandBytes, kChunkBytes);
                    const uint32_t left = min(kBlockK, tile.rows - b * kBlockK);
#pragma unroll
                    for (uint32_t k = 0; k < kBlockK / kUmmaK; ++k)
                        if (k * kUmmaK < left)
                            ptx::mma_bf16_1cta(tmem_d, dd + 128u * k, da + 128u * k, kIdesc, (b | k) != 0u ? 1u : 0u);
                    ptx::mma_commit_1cta(empty_bar(stage));
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok)
                    break;
                ptx::mma_commit_1cta(acc_full_bar(acc));
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            role_ok = ok;
        }
        __syncwarp();
    } else if (warp == 6) {
        // ----------------------------------------------------------- fix warp --
        uint32_t stage = 0;
        uint32_t tail_phase = 0;  // bit s: parity of the next use of tail_bar(s)
        bool ok = true;
        for (uint64_t round = 0, t; ok && (t = dealt_tile(round, cluster, num_clusters)) < num_tiles; ++round) {
            const WgradSplitTile tile = wgrad_split_tile<S>(static_cast<uint32_t>(t), m_blocks, n_blocks, rank, tab);
            if (tile.blocks == 0)
                continue;
            const uint32_t last = (stage + tile.blocks - 1) % STAGES;
            stage = (stage + tile.blocks) % STAGES;
            const uint32_t left = tile.rows - (tile.blocks - 1) * kBlockK;  // 1 .. 64
            if ((left & 15u) == 0u)
                continue;
            ok = wait_bounded(tail_bar(last), (tail_phase >> last) & 1u, ctl, 4);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            tail_phase ^= 1u << last;
            const uint32_t sd = smem_base + last * L::kStageBytes;
            const uint32_t end = (left + 15u) & ~15u;
            for (uint32_t r = left + (lane >> 3); r < end; r += 4) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    ptx::st_shared_v4(sd + j * kChunkBytes + r * 128u + (lane & 7u) * 16u, 0u, 0u, 0u, 0u);
            }
            ptx::fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive(full_bar(last));
            __syncwarp();
        }
        role_ok = ok;
    } else {
        // ----------------------------------------------------------- epilogue --
        const uint32_t quarter = warp & 3u, w = warp - 2u;
        const uint32_t exchange = smem_base + L::kExchangeOffset;
        const uint8_t *from = smem_gen + L::kExchangeOffset + w * L::kWarpBytes + lane * 16u;
        uint32_t acc = 0, acc_phase = 0, parity = 0;
        bool ok = true;
        for (uint64_t round = 0, t; ok && (t = dealt_tile(round, cluster, num_clusters)) < num_tiles; ++round, parity ^= 1u) {
            const WgradSplitTile tile = wgrad_split_tile<S>(static_cast<uint32_t>(t), m_blocks, n_blocks, rank, tab);
            uint32_t v[kWgradSplitTile];  // one row of DW's tile
            if (tile.blocks > 0) {
                ok = wait_bounded(acc_full_bar(acc), acc_phase, ctl, 3);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t taddr = tmem_base + acc * kWgradSplitTile + ((quarter * 32u) << 16);
#pragma unroll
                for (uint32_t c = 0; c < kWgradSplitTile; c += 32) {
                    uint32_t part[32];
                    ptx::tmem_ld_32x32b_x32(taddr + c, part);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i)
                        v[c + i] = part[i];
                }
                ptx::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(acc_empty_bar(acc));
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kWgradSplitTile; ++i)
                    v[i] = 0u;
            }
            // the other CTAs' shares go to them, once they have read what this one sent for its tile before
            ok = wait_bounded<true>(sums_taken_bar, parity ^ 1u, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
#pragma unroll
            for (uint32_t d = 0; d < S; ++d) {
                if (d == rank)
                    continue;
                const uint32_t slot = rank - (rank > d ? 1u : 0u);  // of this CTA among the others of CTA d
                const uint32_t to = ptx::mapa_shared(exchange + slot * L::kPartBytes + w * L::kWarpBytes + lane * 16u, d);
#pragma unroll
                for (uint32_t i = 0; i < L::kShare; i += 4)
                    ptx::st_shared_cluster_v4(to + i * 128u, v[d * L::kShare + i], v[d * L::kShare + i + 1], v[d * L::kShare + i + 2],
                                              v[d * L::kShare + i + 3]);
            }
            __syncwarp();
            if (lane < S && lane != rank)
                ptx::mbar_arrive_cluster_addr(ptx::mapa_shared(sums_full_bar, lane));
            uint32_t mine[L::kShare];
#pragma unroll
            for (uint32_t d = 0; d < S; ++d)
                if (d == rank) {
#pragma unroll
                    for (uint32_t i = 0; i < L::kShare; ++i)
                        mine[i] = v[d * L::kShare + i];
                }
            ok = wait_bounded<true>(sums_full_bar, parity, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            uint32_t out[L::kShare];
#pragma unroll
            for (uint32_t i = 0; i < L::kShare; i += 4) {
                float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t d = 0; d < S; ++d) {
                    float4 part = make_float4(__uint_as_float(mine[i]), __uint_as_float(mine[i + 1]), __uint_as_float(mine[i + 2]),
                                              __uint_as_float(mine[i + 3]));
                    if (d != rank)
                        part = *reinterpret_cast<const float4 *>(from + (d - (d > rank ? 1u : 0u)) * L::kPartBytes + i * 128u);
                    total.x += part.x, total.y += part.y, total.z += part.z, total.w += part.w;
                }
                out[i] = __float_as_uint(total.x), out[i + 1] = __float_as_uint(total.y);
                out[i + 2] = __float_as_uint(total.z), out[i + 3] = __float_as_uint(total.w);
            }
            __syncwarp();
            // what came for this warp has been read: its place serves as staging buffer
            GemmParams q{};
            q.c = p.c + static_cast<uint64_t>(tile.group) * p.c_stride;
            q.ldc = p.ldc;
            q.m = p.n;
            q.c_vec_ok = p.c_vec_ok;
            const uint32_t row0 = tile.m0 + quarter * 32u, col = tile.n0 + rank * L::kShare;
            if (row0 < p.n && col < p.k)
                store_share<L::kShare>(q, exchange + w * L::kWarpBytes, lane, row0, col, p.k, out);
            __syncwarp();
            if (lane < S && lane != rank)
                ptx::mbar_arrive_cluster_addr(ptx::mapa_shared(sums_taken_bar, lane));
        }
        role_ok = ok;
    }
    if (!role_ok) {
        // tell the other CTAs, so that their roles stop waiting on us
        for (uint32_t d = 0; d < S; ++d)
            if (d != rank)
                ptx::st_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(const_cast<int *>(abort_flag)), d), 1u);
    }

    // ---------------------------------------------------------------- teardown --
    __syncwarp();
    ptx::tcgen05_fence_before();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (warp == 1) {
        if (*abort_flag) {
            for (int i = 0; i < 256; ++i)
                __nanosleep(1000);
        }
        ptx::tcgen05_fence_after();
        ptx::tmem_dealloc_1cta(tmem_base, kTmemCols);
    }
}

}  // namespace maize
