// The grouped product where the tiles are too few to fill the SMs (a few rows left for a few experts, a long K): a cluster of
// S = 2, 4 or 8 CTAs shares a tile and splits K.
//
// As in gemm_sm100_grouped.cuh the weights are the M side of the MMA (128 rows of W per tile) and the rows of A its N side (up
// to 64 per tile).  Each CTA of the cluster accumulates its part of the k-blocks in its own tensor memory; the parts meet in
// distributed shared memory: every CTA finishes the tile's rows of A that are its share (64 / S), adds the S parts of them in
// the order of K, rounds once and stores.  No global scratch, a fixed order of sums.
//
// Bound: the latency of one CTA's k-blocks, about 0.3 us each; eight rows for five experts, 144 x 6936: 8 us instead of 35.
#pragma once
#include "gemm_sm100_grouped.cuh"

namespace maize {

constexpr uint32_t kSplitTileRows = 64;   // rows of A per tile at most
constexpr uint32_t kSplitTileCols = 128;  // columns of C per tile
constexpr uint32_t kSplitRowUnit = 16;    // the MMA's N for 128 M-side rows

template <uint32_t S, uint32_t STAGES>
struct GroupedSplitLayout {
    static constexpr uint32_t kShare = kSplitTileRows / S;  // rows of A that one CTA finishes
    static constexpr uint32_t kWBytes = kSplitTileCols * kBlockK * 2;
    static constexpr uint32_t kABytes = kSplitTileRows * kBlockK * 2;
    static constexpr uint32_t kStageBytes = kWBytes + kABytes;
    static constexpr uint32_t kExchangeOffset = STAGES * kStageBytes;  // from each other CTA: [row of A][column of C]
    static constexpr uint32_t kPartBytes = kShare * kSplitTileCols * 4;
    static constexpr uint32_t kBarOffset = kExchangeOffset + (S - 1) * kPartBytes;
    static constexpr uint32_t kNumBars = 2 * STAGES + 4 + 2;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kTableOffset = (kAbortOffset + 4 + 15) / 16 * 16;
    static constexpr uint32_t kUsedBytes = kTableOffset + kGroupTableBytes;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
};

// W_KN: the weights are stored K x N, two boxes of {64 columns, 64 k-rows} per k-block, read as an MN-major operand.
template <bool W_KN, uint32_t S, uint32_t STAGES>
__global__ void __launch_bounds__(kNumThreads, 1)
gemm_bf16_sm100_grouped_split(const __grid_constant__ RowMaps tma_a, const __grid_constant__ CUtensorMap tma_w,
                              const GroupedParams p)
{
    using L = GroupedSplitLayout<S, STAGES>;
    constexpr uint32_t kTmemCols = 2 * kSplitTileRows;  // two accumulator buffers
    constexpr uint32_t kChunkBytes = kBlockK * 128;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    const uint32_t sums_full_bar = bar_base + 8u * (2 * STAGES + 4);   // the other CTAs' sums are here
    const uint32_t sums_taken_bar = bar_base + 8u * (2 * STAGES + 5);  // the others have read what this CTA sent
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);
    const GroupTable tab(smem_gen + L::kTableOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t rank = ptx::cluster_cta_rank();
    const uint32_t cluster = blockIdx.x / S;
    const uint32_t num_clusters = gridDim.x / S;
    const uint32_t all_kb = (p.k + kBlockK - 1) / kBlockK;
    const uint32_t per_cta = (all_kb + S - 1) / S;
    const uint32_t kb0 = min(rank * per_cta, all_kb);
    const uint32_t num_kb = min(per_cta, all_kb - kb0);  // may be 0 in the last CTAs
    const uint32_t n_blocks = (p.n + kSplitTileCols - 1) / kSplitTileCols;
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_w);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
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
    // all CTAs of a cluster read the same offsets and come to the same tiles
    uint32_t row_tiles = 0;
    build_group_table<kSplitTileRows>(p, tab, row_tiles);
    const uint64_t num_tiles = static_cast<uint64_t>(row_tiles) * n_blocks;

    bool role_ok = true;
    if (warp == 0) {
        // ------------------------------------------------------- TMA producer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, g = 0;
            bool ok = true;
            for (uint64_t t = cluster; ok && t < num_tiles; t += num_clusters) {
                const GroupedTile tile = grouped_tile<kSplitRowUnit>(t, n_blocks, tab, g);
                const uint32_t box = tile.rows <= 16 ? 0u : (tile.rows <= 32 ? 1u : 2u);
                const uint32_t bytes = L::kWBytes + (16u << box) * (kBlockK * 2);
                const int32_t n0 = static_cast<int32_t>(tile.n_blk * kSplitTileCols), r0 = static_cast<int32_t>(tile.row0);
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = wait_bounded(empty_bar(stage), phase ^ 1u, ctl, 1);
                    if (!ok)
                        break;
                    const uint32_t sw = smem_base + stage * L::kStageBytes;
                    const int32_t kx = static_cast<int32_t>((kb0 + kb) * kBlockK);
                    ptx::mbar_arrive_expect_tx(full_bar(stage), bytes);
                    if constexpr (W_KN) {
#pragma unroll
                        for (uint32_t j = 0; j < 2; ++j)
                            ptx::tma_load_3d(sw + j * kChunkBytes, &tma_w, full_bar(stage), n0 + static_cast<int32_t>(64u * j), kx,
                                             static_cast<int32_t>(tile.group));
                    } else {
                        ptx::tma_load_3d(sw, &tma_w, full_bar(stage), kx, n0, static_cast<int32_t>(tile.group));
                    }
                    ptx::tma_load_2d(sw + L::kWBytes, &tma_a.box[box], full_bar(stage), kx, r0);
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
        if (lane == 0 && num_kb > 0) {
            uint32_t stage = 0, phase = 0, g = 0;
            uint32_t acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint64_t t = cluster; ok && t < num_tiles; t += num_clusters) {
                const GroupedTile tile = grouped_tile<kSplitRowUnit>(t, n_blocks, tab, g);
                const uint32_t mma_n = (tile.rows + kSplitRowUnit - 1) / kSplitRowUnit * kSplitRowUnit;
                const uint32_t idesc = ptx::make_instr_desc_bf16(kBlockM, mma_n, false, W_KN);
                ok = wait_bounded(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t tmem_d = tmem_base + acc * kSplitTileRows;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = wait_bounded(full_bar(stage), phase, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sw = smem_base + stage * L::kStageBytes;
                    const uint64_t dw = W_KN ? ptx::make_smem_desc_sw128_mn(sw, kChunkBytes) : ptx::make_smem_desc_sw128(sw);
                    const uint64_t da = ptx::make_smem_desc_sw128(sw + L::kWBytes);
                    constexpr uint32_t kStepW = W_KN ? 128u : 2u;
#pragma unroll
                    for (uint32_t k = 0; k < kBlockK / kUmmaK; ++k)
                        ptx::mma_bf16_1cta(tmem_d, dw + kStepW * k, da + 2u * k, idesc, (kb | k) != 0u ? 1u : 0u);
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
    } else {
        // ----------------------------------------------------------- epilogue --
        const uint32_t quarter = warp & 3u;
        const uint32_t my_col = quarter * 32u + lane;  // of the tile
        const uint32_t exchange = smem_base + L::kExchangeOffset;
        const float *from = reinterpret_cast<const float *>(smem_gen + L::kExchangeOffset) + my_col;
        uint32_t acc = 0, acc_phase = 0, g = 0, parity = 0;
        bool ok = true;
        for (uint64_t t = cluster; ok && t < num_tiles; t += num_clusters, parity ^= 1u) {
            const GroupedTile tile = grouped_tile<kSplitRowUnit>(t, n_blocks, tab, g);
            uint32_t v[kSplitTileRows];  // one column of C, a register per row of A
#pragma unroll
            for (uint32_t i = 0; i < kSplitTileRows; ++i)
                v[i] = 0u;
            if (num_kb > 0) {
                ok = wait_bounded(acc_full_bar(acc), acc_phase, ctl, 3);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t taddr = tmem_base + acc * kSplitTileRows + ((quarter * 32u) << 16);
                uint32_t lo[32], hi[32];
                ptx::tmem_ld_32x32b_x32(taddr, lo);
                if (tile.rows > 32)
                    ptx::tmem_ld_32x32b_x32(taddr + 32u, hi);
                ptx::tmem_ld_wait();
                ptx::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(acc_empty_bar(acc));
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) {
                    v[i] = lo[i];
                    if (tile.rows > 32)
                        v[32 + i] = hi[i];
                }
            }
            // the other CTAs' shares go to them, once they have read what this one sent for its tile before
            ok = wait_bounded<true>(sums_taken_bar, parity ^ 1u, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
#pragma unroll
            for (uint32_t d = 0; d < S; ++d) {
                if (d == rank || d * L::kShare >= tile.rows)
                    continue;
                const uint32_t slot = rank - (rank > d ? 1u : 0u);  // of this CTA among the others of CTA d
                const uint32_t to = ptx::mapa_shared(exchange + slot * L::kPartBytes + my_col * 4u, d);
#pragma unroll
                for (uint32_t i = 0; i < L::kShare; ++i)
                    ptx::st_shared_cluster_u32(to + i * (kSplitTileCols * 4u), v[d * L::kShare + i]);
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
            uint32_t out[32];
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i)
                out[i] = 0u;
            const uint32_t first = rank * L::kShare;  // of the tile's rows
            if (first < tile.rows) {
#pragma unroll
                for (uint32_t i = 0; i < L::kShare; ++i) {
                    float total = 0.0f;
#pragma unroll
                    for (uint32_t d = 0; d < S; ++d)
                        total += d == rank ? __uint_as_float(mine[i])
                                           : from[(d - (d > rank ? 1u : 0u)) * (L::kPartBytes / 4) + i * kSplitTileCols];
                    out[i] = __float_as_uint(total);
                }
            }
            __syncwarp();
            if (lane < S && lane != rank)
                ptx::mbar_arrive_cluster_addr(ptx::mapa_shared(sums_taken_bar, lane));
            const uint32_t warp_col = tile.n_blk * kSplitTileCols + quarter * 32u;
            if (first < tile.rows && warp_col < p.n)
                store_transposed_chunk(p, tile.row0 + first, min(L::kShare, tile.rows - first), warp_col + lane, lane, out);
            __syncwarp();
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
