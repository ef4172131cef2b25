// Weight gradient of the grouped product: for every group g, over its rows r = offsets[g] .. offsets[g+1]-1,
//
//     DW[g] (N x K) = sum_r  DC[r, :]^T  A[r, :]        (a group without rows: zeros)
//
// The reduction runs over the ROWS, so both operands are MN-major: a k-block is 64 rows, loaded as boxes of
// {64 columns, 64 rows} of DC (the MMA's M side, 256 columns per CTA pair) and of A (its N side).
//
// A group ends at any row, and a box that crosses its end brings in rows of the next group.  They must not take part, and
// multiplying them by zeros on one side would not do (0 * Inf = NaN), so they are cleared on both sides: the last k-block
// of a group with `v` rows left issues only ceil(v / 16) of its four MMAs, and if v is no multiple of 16 a "fix" warp of
// each CTA waits for that block's bytes, overwrites rows v .. of the last 16 in shared memory with zeros, orders the
// writes before the tensor core's reads (fence.proxy.async) and only then lets the MMA thread have the stage.  With
// MN-major tiles a row is 128 consecutive bytes per box whatever the swizzle does inside it, so the clearing is a plain
// fill of at most 15 rows x 4 boxes x 128 bytes.
//
// Roles per CTA: TMA producer, MMA issuer (leader only), eight epilogue warps, the fix warp.
// Bound: tensor pipe where groups have two thousand rows (8 x 2048, 4096 x 4096: 379 us, 1.45 PFLOP/s); below, what a tile costs
// beside its sum (16 x 512, 4096 x 2048: 148 us, 113 without the stores of DW).
#pragma once
#include "gemm_sm100_grouped.cuh"

namespace maize {

// Eight epilogue warps, two for each quarter of the lanes, that take the tile's groups of 64 columns in turn.
constexpr uint32_t kWgradEpilogueWarps = 8;
constexpr uint32_t kWgradFixWarp = 2 + kWgradEpilogueWarps;
constexpr uint32_t kWgradThreads = 32 * (kWgradFixWarp + 1);
// One staging buffer of 32 rows x 64 columns per warp (a second one, at the cost of a ring stage, lost: 16 uneven groups of 8192
// rows, 4096 x 2048, 146 us instead of 136).
constexpr uint32_t kWgradStageWarpBytes = kTmaStoreBufBytes;

template <uint32_t STAGES>
struct WgradSmemLayout {
    static constexpr uint32_t kOperandBytes = kBlockM * kBlockK * 2;  // two boxes of 64 columns x 64 rows
    static constexpr uint32_t kStageBytes = 2 * kOperandBytes;        // [DC0, DC1, A0, A1]
    static constexpr uint32_t kStagingOffset = STAGES * kStageBytes;
    static constexpr uint32_t kBarOffset = kStagingOffset + kWgradEpilogueWarps * kWgradStageWarpBytes;
    static constexpr uint32_t kNumBars = 4 * STAGES + 4;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kTableOffset = (kAbortOffset + 4 + 15) / 16 * 16;
    static constexpr uint32_t kUsedBytes = kTableOffset + kGroupTableBytes;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
};

struct WgradTile {
    uint32_t group, m_blk, n_blk, row0, rows, steps;
};

constexpr uint32_t kGroupMaxClasses = 128;  // of sort_groups, which counts them in `first`
static_assert(kGroupMaxClasses <= kGroupedMaxGroups, "table of groups");

// Whole CTA.  Sets t.order to the groups by ascending class_of(rows of the group), equal ones in their own order: a counting
// sort, the same in every CTA.  class_of is below kGroupMaxClasses.
template <typename ClassOf>
__device__ __forceinline__ void sort_groups(const GroupedParams &p, const GroupTable &t, ClassOf class_of)
{
    auto class_at = [&](uint32_t g) { return class_of(t.offset[g + 1] - t.offset[g]); };
    for (uint32_t i = threadIdx.x; i < kGroupMaxClasses; i += blockDim.x)
        t.first[i] = 0;
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < p.groups; g += blockDim.x)
        atomicAdd(&t.first[class_at(g)], 1u);
    __syncthreads();
    if (threadIdx.x < 32) {
        uint32_t total = 0;
#pragma unroll
        for (uint32_t base = 0; base < kGroupMaxClasses; base += 32) {
            const uint32_t mine = t.first[base + threadIdx.x];
            uint32_t sum = mine;
#pragma unroll
            for (uint32_t d = 1; d < 32; d <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, sum, d);
                if (threadIdx.x >= d)
                    sum += up;
            }
            t.first[base + threadIdx.x] = total + sum - mine;
            total += __shfl_sync(0xffffffffu, sum, 31);
        }
        __syncwarp();
        for (uint32_t base = 0; base < p.groups; base += 32) {
            const uint32_t g = base + threadIdx.x;
            const uint32_t cls = g < p.groups ? class_at(g) : kGroupMaxClasses;
            const uint32_t same = __match_any_sync(0xffffffffu, cls);
            const uint32_t before = __popc(same & ((1u << threadIdx.x) - 1u));
            uint32_t place = 0;
            if (g < p.groups) {
                place = t.first[cls] + before;
                t.order[place] = static_cast<uint16_t>(g);
            }
            __syncwarp();
            if (g < p.groups && before == 0)
                t.first[cls] = place + __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
}

// The tile of a launch that pair (cluster) `pair` works on in round `round`: one round from left to right, the next from right to
// left, so that pairs which got the longer tiles of one round get the shorter ones of the next.  With the longest groups first:
// 24 uneven groups of 6263 rows in all, 896 x 352, 16.9 -> 15.4 us.
__device__ __forceinline__ uint64_t dealt_tile(uint64_t round, uint32_t pair, uint32_t num_pairs)
{
    return round * num_pairs + ((round & 1u) != 0u ? num_pairs - 1u - pair : pair);
}

// Whole CTA.  Reads the offsets into shared memory and, if the tiles take more than one round, orders the groups, those with the
// most rows first: by the number of 64-row blocks, four classes to a doubling.  (In one round no order matters, and sorting
// costs 0.7 us: 3 rows of 4 groups, 512 x 256, 6.6 instead of 5.9.)  False if the offsets are not right.
__device__ __forceinline__ bool build_wgrad_table(const GroupedParams &p, const GroupTable &t, bool one_round)
{
    if (one_round)
        for (uint32_t g = threadIdx.x; g < p.groups; g += blockDim.x)
            t.order[g] = static_cast<uint16_t>(g);
    if (!load_offsets(p, t.offset))
        return false;
    if (!one_round)
        sort_groups(p, t, [](uint32_t rows) {
            if (rows == 0)
                return kGroupMaxClasses - 1u;
            const uint32_t blocks = (rows + kBlockK - 1) / kBlockK, log2 = 31u - __clz(blocks);
            return kGroupMaxClasses - 2u - (log2 * 4u + ((blocks << 2 >> log2) & 3u));
        });
    return true;
}

// Tiles of one group follow each other; within it the blocks of A's columns run fastest.
__device__ __forceinline__ WgradTile wgrad_tile(uint32_t t, uint32_t m_blocks, uint32_t n_blocks, const GroupTable &tab)
{
    const uint32_t per_group = m_blocks * n_blocks;
    WgradTile r;
    const uint32_t at = t / per_group, local = t - at * per_group;
    r.group = tab.order[at];
    r.m_blk = local / n_blocks;
    r.n_blk = local - r.m_blk * n_blocks;
    r.row0 = tab.offset[r.group];
    r.rows = tab.offset[r.group + 1] - r.row0;
    r.steps = (r.rows + kBlockK - 1) / kBlockK;
    return r;
}

// Drains this warp's 32 x 256 part of the accumulator (or writes zeros) through shared memory and TMA stores of 32 x 64
// boxes into matrix `z` of the stack; the map clips at N and K.  `loaded` is called once, when the last of it is in registers.
template <typename Loaded>
__device__ __forceinline__ void wgrad_drain_tma(const GroupedParams &p, const CUtensorMap *tma_c, uint32_t stage_u32,
                                                uint32_t taddr, bool zeros, uint32_t lane, uint32_t row0, uint32_t col0,
                                                uint32_t z, uint32_t turn, Loaded loaded)
{
    // groups of 64 columns that K has in this tile, as far as this warp's rows exist
    const uint32_t groups = row0 >= p.n ? 0u : min(kGroupedTileCols / 64u, (p.k - col0 + 63u) / 64u);
    if (turn >= groups)
        loaded();
#pragma unroll 1
    for (uint32_t g = turn; g < groups; g += 2) {
        const uint32_t col = col0 + g * 64u;
        uint32_t v0[32], v1[32];
        if (zeros) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v0[i] = v1[i] = 0u;
        } else {
            ptx::tmem_ld_32x32b_x32(taddr + g * 64u, v0);
            ptx::tmem_ld_32x32b_x32(taddr + g * 64u + 32u, v1);
            ptx::tmem_ld_wait();
        }
        if (g + 2 >= groups)
            loaded();
        if (lane == 0)
            ptx::bulk_wait_group_read<0>();  // the buffer's last store has read it
        __syncwarp();
        const uint32_t row = stage_u32 + lane * 128u;
        const uint32_t sw = lane & 7u;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            ptx::st_shared_v4(row + ((j ^ sw) << 4), ptx::pack_bf16x2(v0[8 * j], v0[8 * j + 1]),
                              ptx::pack_bf16x2(v0[8 * j + 2], v0[8 * j + 3]), ptx::pack_bf16x2(v0[8 * j + 4], v0[8 * j + 5]),
                              ptx::pack_bf16x2(v0[8 * j + 6], v0[8 * j + 7]));
            ptx::st_shared_v4(row + (((j + 4u) ^ sw) << 4), ptx::pack_bf16x2(v1[8 * j], v1[8 * j + 1]),
                              ptx::pack_bf16x2(v1[8 * j + 2], v1[8 * j + 3]), ptx::pack_bf16x2(v1[8 * j + 4], v1[8 * j + 5]),
                              ptx::pack_bf16x2(v1[8 * j + 6], v1[8 * j + 7]));
        }
        ptx::fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
            // DW passes through L2 once: evict first (32 groups of 128 rows, 1024 x 1408: 47 -> 41 us)
            if (p.c_evict_first)
                ptx::tma_store_3d_hint(tma_c, stage_u32, static_cast<int32_t>(col), static_cast<int32_t>(row0), static_cast<int32_t>(z),
                                       ptx::policy_evict_first());
            else
                ptx::tma_store_3d(tma_c, stage_u32, static_cast<int32_t>(col), static_cast<int32_t>(row0), static_cast<int32_t>(z));
            ptx::bulk_commit_group();
        }
    }
}

// The same with plain stores, for a DW whose rows are not 16-byte aligned: lane = row, 2-byte stores that are
// consecutive across the warp after a transposition through the warp's staging buffer.
template <typename Loaded>
__device__ __forceinline__ void wgrad_drain_plain(const GroupedParams &p, uint8_t *stage_warp, uint32_t taddr, bool zeros,
                                                  uint32_t lane, uint32_t row0, uint32_t col0, uint32_t z,
                                                  uint32_t turn, Loaded loaded)
{
    GemmParams q{};
    q.c = p.c + static_cast<uint64_t>(z) * p.c_stride;
    q.ldc = p.ldc;
    q.m = p.n;
    q.n = p.k;
    q.c_vec_ok = 0;
#pragma unroll 1
    for (uint32_t c = turn; c < kGroupedTileCols / 32; c += 2) {
        uint32_t v[32];
        if (zeros) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[i] = 0u;
        } else {
            ptx::tmem_ld_32x32b_x32(taddr + c * 32u, v);
            ptx::tmem_ld_wait();
        }
        if (c + 2 >= kGroupedTileCols / 32)
            loaded();
        store_chunk(q, stage_warp, row0, col0 + c * 32u, lane, v);
        __syncwarp();
    }
}

template <uint32_t STAGES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWgradThreads, 1)
gemm_bf16_sm100_grouped_wgrad(const __grid_constant__ CUtensorMap tma_dc, const __grid_constant__ CUtensorMap tma_a,
                              const __grid_constant__ CUtensorMap tma_dw, const GroupedParams p)
{
    using L = WgradSmemLayout<STAGES>;
    constexpr uint32_t kTmemCols = 2 * kGroupedTileCols;
    constexpr uint32_t kChunkBytes = kBlockK * 128;
    constexpr uint32_t kIdesc = ptx::make_instr_desc_bf16(2 * kBlockM, kGroupedTileCols, true, true);

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    auto tail_bar = [&](uint32_t s) { return bar_base + 8u * (2 * STAGES + 4 + s); };  // this CTA's bytes of a cut block
    auto peer_bar = [&](uint32_t s) { return bar_base + 8u * (3 * STAGES + 4 + s); };  // leader: the peer's cut block is clear
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);
    const GroupTable tab(smem_gen + L::kTableOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t cta_rank = ptx::cluster_cta_rank();
    const uint32_t pair = blockIdx.x >> 1;
    const uint32_t num_pairs = gridDim.x >> 1;
    const uint32_t m_blocks = (p.n + 2 * kBlockM - 1) / (2 * kBlockM);
    const uint32_t n_blocks = (p.k + kGroupedTileCols - 1) / kGroupedTileCols;
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_dc);
        ptx::prefetch_tensormap(&tma_a);
        if (p.c_tma_ok)
            ptx::prefetch_tensormap(&tma_dw);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);   // the leader's producer and the bytes of both CTAs, or the leader's fix warp
            ptx::mbar_init(empty_bar(s), 1);  // one tcgen05.commit of the leader
            ptx::mbar_init(tail_bar(s), 1);   // this CTA's producer and its bytes
            ptx::mbar_init(peer_bar(s), 1);   // the peer's fix warp
        }
        for (uint32_t b = 0; b < 2; ++b) {
            ptx::mbar_init(acc_full_bar(b), 1);
            ptx::mbar_init(acc_empty_bar(b), 2 * kWgradEpilogueWarps);
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc_2cta(ptx::smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemCols);
        ptx::tmem_relinquish_2cta();
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
    const uint32_t num_tiles = build_wgrad_table(p, tab, all_tiles <= num_pairs) ? all_tiles : 0u;

    bool role_ok = true;
    if (warp == 0) {
        // ------------------------------------------------------- TMA producer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint64_t round = 0, t; ok && (t = dealt_tile(round, pair, num_pairs)) < num_tiles; ++round) {
                const WgradTile tile = wgrad_tile(static_cast<uint32_t>(t), m_blocks, n_blocks, tab);
                const int32_t n0 = static_cast<int32_t>(tile.m_blk * 2 * kBlockM + cta_rank * kBlockM);
                const int32_t k0 = static_cast<int32_t>(tile.n_blk * kGroupedTileCols + cta_rank * kBlockM);
                for (uint32_t step = 0; step < tile.steps; ++step) {
                    ok = wait_bounded<true>(empty_bar(stage), phase ^ 1u, ctl, 1);
                    if (!ok)
                        break;
                    const uint32_t sd = smem_base + stage * L::kStageBytes;
                    const uint32_t sa = sd + L::kOperandBytes;
                    const int32_t r = static_cast<int32_t>(tile.row0 + step * kBlockK);
                    const uint32_t left = tile.rows - step * kBlockK;
                    if (left < kBlockK && (left & 15u) != 0u) {
                        // a cut block: its bytes go to this CTA's own barrier, the fix warp passes the stage on
                        ptx::mbar_arrive_expect_tx(tail_bar(stage), L::kStageBytes);
#pragma unroll
                        for (uint32_t j = 0; j < 2; ++j) {
                            ptx::tma_load_2d(sd + j * kChunkBytes, &tma_dc, tail_bar(stage), n0 + static_cast<int32_t>(64u * j), r);
                            ptx::tma_load_2d(sa + j * kChunkBytes, &tma_a, tail_bar(stage), k0 + static_cast<int32_t>(64u * j), r);
                        }
                    } else {
                        const uint32_t leader_full = ptx::mapa_shared(full_bar(stage), 0);
                        if (cta_rank == 0)
                            ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * L::kStageBytes);
#pragma unroll
                        for (uint32_t j = 0; j < 2; ++j) {
                            ptx::tma_load_2d_pair(sd + j * kChunkBytes, &tma_dc, leader_full, n0 + static_cast<int32_t>(64u * j), r);
                            ptx::tma_load_2d_pair(sa + j * kChunkBytes, &tma_a, leader_full, k0 + static_cast<int32_t>(64u * j), r);
                        }
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
        // ------------------------------------------- MMA issuer (leader only) --
        if (lane == 0 && cta_rank == 0) {
            uint32_t stage = 0, phase = 0;
            uint32_t acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint64_t round = 0, t; ok && (t = dealt_tile(round, pair, num_pairs)) < num_tiles; ++round) {
                const WgradTile tile = wgrad_tile(static_cast<uint32_t>(t), m_blocks, n_blocks, tab);
                if (tile.steps == 0)
                    continue;  // no rows: the epilogue writes zeros, no accumulator changes hands
                ok = wait_bounded<true>(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t tmem_d = tmem_base + acc * kGroupedTileCols;
                for (uint32_t step = 0; step < tile.steps; ++step) {
                    ok = wait_bounded<true>(full_bar(stage), phase, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sd = smem_base + stage * L::kStageBytes;
                    const uint64_t dd = ptx::make_smem_desc_sw128_mn(sd, kChunkBytes);
                    const uint64_t da = ptx::make_smem_desc_sw128_mn(sd + L::kOperandBytes, kChunkBytes);
                    const uint32_t left = min(kBlockK, tile.rows - step * kBlockK);
#pragma unroll
                    for (uint32_t k = 0; k < kBlockK / kUmmaK; ++k)
                        if (k * kUmmaK < left)
                            ptx::mma_bf16_2cta(tmem_d, dd + 128u * k, da + 128u * k, kIdesc, (step | k) != 0u ? 1u : 0u);
                    ptx::mma_commit_2cta_mask(empty_bar(stage), 3);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok)
                    break;
                ptx::mma_commit_2cta_mask(acc_full_bar(acc), 3);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            role_ok = ok;
        }
        __syncwarp();
    } else if (warp == kWgradFixWarp) {
        // ----------------------------------------------------------- fix warp --
        uint32_t stage = 0;
        uint32_t tail_phase = 0;  // bit s: parity of the next use of tail_bar(s) and peer_bar(s)
        bool ok = true;
        for (uint64_t round = 0, t; ok && (t = dealt_tile(round, pair, num_pairs)) < num_tiles; ++round) {
            const WgradTile tile = wgrad_tile(static_cast<uint32_t>(t), m_blocks, n_blocks, tab);
            if (tile.steps == 0)
                continue;
            const uint32_t last = (stage + tile.steps - 1) % STAGES;
            stage = (stage + tile.steps) % STAGES;
            const uint32_t left = tile.rows - (tile.steps - 1) * kBlockK;  // 1 .. 64
            if ((left & 15u) == 0u)
                continue;
            ok = wait_bounded<true>(tail_bar(last), (tail_phase >> last) & 1u, ctl, 4);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            const uint32_t sd = smem_base + last * L::kStageBytes;
            const uint32_t end = (left + 15u) & ~15u;
            // 8 lanes clear a 128-byte row, 4 rows at a time, in the four boxes of the stage
            for (uint32_t r = left + (lane >> 3); r < end; r += 4) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    ptx::st_shared_v4(sd + j * kChunkBytes + r * 128u + (lane & 7u) * 16u, 0u, 0u, 0u, 0u);
            }
            ptx::fence_proxy_async_shared();
            __syncwarp();
            // The peer tells the leader's fix warp and that one the MMA thread.  (An arrival of the peer's producer on
            // every stage instead, so that the stage's barrier itself counts both CTAs, cost two thirds of the rate: a
            // remote arrival releases at cluster scope, and the loads behind it wait for that.)
            if (cta_rank != 0) {
                if (lane == 0)
                    ptx::mbar_arrive_cluster_addr(ptx::mapa_shared(peer_bar(last), 0));
            } else {
                ok = wait_bounded<true>(peer_bar(last), (tail_phase >> last) & 1u, ctl, 4);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok)
                    break;
                if (lane == 0)
                    ptx::mbar_arrive(full_bar(last));
            }
            tail_phase ^= 1u << last;
            __syncwarp();
        }
        role_ok = ok;
    } else {
        // ----------------------------------------------------------- epilogue --
        const uint32_t quarter = warp & 3u, turn = (warp - 2u) >> 2;
        uint8_t *stage_warp = smem_gen + L::kStagingOffset + (warp - 2u) * kWgradStageWarpBytes;
        const uint32_t stage_u32 = smem_base + L::kStagingOffset + (warp - 2u) * kWgradStageWarpBytes;
        uint32_t acc = 0, acc_phase = 0;
        bool ok = true;
        for (uint64_t round = 0, t; ok && (t = dealt_tile(round, pair, num_pairs)) < num_tiles; ++round) {
            const WgradTile tile = wgrad_tile(static_cast<uint32_t>(t), m_blocks, n_blocks, tab);
            const bool zeros = tile.steps == 0;
            if (!zeros) {
                ok = wait_bounded<true>(acc_full_bar(acc), acc_phase, ctl, 3);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
            }
            const uint32_t taddr = tmem_base + acc * kGroupedTileCols + ((quarter * 32u) << 16);
            const uint32_t row0 = tile.m_blk * 2 * kBlockM + cta_rank * kBlockM + quarter * 32u;
            const uint32_t col0 = tile.n_blk * kGroupedTileCols;
            // The accumulator goes back as soon as it is in registers, without a release: the loads are complete, and a release
            // at cluster scope would wait for the warp's stores, 3300 cycles a
            // tile (16 uneven groups of 2000 rows in all, 2048 x 2048: 42 -> 33 us; 64 of 8192, 2048 x 1024: 94 -> 75).
            auto hand_back = [&] {
                if (zeros)
                    return;
                ptx::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive_cluster_addr_relaxed(ptx::mapa_shared(acc_empty_bar(acc), 0));
            };
            if (p.c_tma_ok)
                wgrad_drain_tma(p, &tma_dw, stage_u32, taddr, zeros, lane, row0, col0, tile.group, turn, hand_back);
            else
                wgrad_drain_plain(p, stage_warp, taddr, zeros, lane, row0, col0, tile.group, turn, hand_back);
            if (!zeros) {
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
        if (p.c_tma_ok)
            tma_store_drain(lane);
        role_ok = ok;
    }
    if (!role_ok)
        ptx::st_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(const_cast<int *>(abort_flag)), cta_rank ^ 1u), 1u);

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
        ptx::tmem_dealloc_2cta(tmem_base, kTmemCols);
    }
}

}  // namespace maize
