// The e4m3 product for few rows of A, or few tiles: K is split over the CTAs of a cluster.  For M <= 128 bound by reading B once.
//
// Rows of A are the M side of the MMA, up to 256 rows of B its N side: a k-block costs a CTA about 0.34 us in MMA issue and
// hand-overs whatever the tile's width, so the operand that streams belongs on the side that may be 256 wide.  16 x 16384 x
// 4096: 16.6 us with B on the M side, 128 rows at a time, 11.9 this way (both with B in L2; 15.2, 4.5 TB/s, when it comes from
// HBM).  For M <= 32 (64) the rows of A are loaded four times (twice)
// into the 128 lanes, so that every promotion warp has lanes with all rows and only some of the columns: REPL copies.  Only
// the m rows there are are loaded (a box that reaches past the end of A takes longer: one row took 16.6 us, 16 rows 13.8);
// what lies in the other lanes is never stored.  For 64 < M the tile is 128 wide, so that four accumulator buffers fit and
// the MMA does not wait for hand-overs.
//
// A cluster of S = 2 or 4 CTAs shares a tile and splits K: each promotes the k-blocks of its part in registers (lane = row
// of A, one register per row of B), then sends every other CTA the sums of that CTA's share of the columns through distributed
// shared memory; each adds its share in the order of the parts, rounds once and stores.  No global scratch, a fixed order.
// (Eight parts lost more in the exchange and in clusters that do not fit beside each other than they gained.)
//
// The kernels with one or two copies need more than the 168 registers that ten warps leave them and spill 236 to 244 bytes; those with
// four take 148.
//
// The host picks the tile's width so that the tiles fill whole rounds of clusters (16384 rows over 74 pairs: one round of
// 224).  The columns of a warp lie in at most two scale blocks of B, each chunk of 32 in one.
#pragma once
#include "gemm_e4m3_sm100.cuh"

namespace maize {

constexpr uint32_t kF8SkinnyThreads = 64 + 32 * 8;

struct F8SkinnyParams {
    GemmParams g;  // C and the sizes; tiles_m blocks of 128 rows of A (1 with copies of them), tiles_n blocks of B
    const float *sa, *sb;
    uint64_t ld_sa, ld_sb;
    uint32_t bn;  // rows of B per tile, a multiple of 32, at most 256
};

template <uint32_t REPL, uint32_t S, uint32_t STAGES>
struct F8SkinnyLayout {
    static_assert(REPL == 1 || REPL == 2 || REPL == 4, "copies of the rows of A");
    static constexpr uint32_t kRows = 128 / REPL;                       // rows of A
    static constexpr uint32_t kWarps = 8;                               // promotion warps, two per quarter of the lanes
    static constexpr uint32_t kTileCols = REPL == 1 ? 128 : 256;        // rows of B per tile at most
    static constexpr uint32_t kBuffers = 512 / kTileCols;               // accumulator buffers that fill tensor memory
    static constexpr uint32_t kWarpCols = REPL == 4 ? 32 : 64;
    static constexpr uint32_t kShare = kWarpCols / S;                   // columns of a warp that one CTA finishes
    static constexpr uint32_t kABytes = kBlockM * kF8BlockK;
    static constexpr uint32_t kBBytes = kTileCols * kF8BlockK;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr uint32_t kExchangeOffset = STAGES * kStageBytes;   // from each other CTA: [warp][4 columns][lane]
    static constexpr uint32_t kPartBytes = kWarps * kShare * 32 * 4;
    static constexpr uint32_t kExchangeBytes = (S - 1) * kPartBytes;
    static constexpr uint32_t kBarOffset = kExchangeOffset + kExchangeBytes;
    static constexpr uint32_t kNumBars = 2 * STAGES + 2 * kBuffers + 2;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kUsedBytes = kAbortOffset + 4;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
    static_assert(kShare >= 8 && kShare <= 32, "columns of a warp that one CTA finishes");
};

template <uint32_t REPL, uint32_t S, uint32_t STAGES>
__global__ void __launch_bounds__(kF8SkinnyThreads, 1)
gemm_e4m3_sm100_skinny(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                       const F8SkinnyParams f)
{
    using L = F8SkinnyLayout<REPL, S, STAGES>;
    constexpr uint32_t kTmemCols = 512;
    constexpr uint32_t kChunks = L::kWarpCols / 32;
    const GemmParams &p = f.g;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + L::kBuffers + b); };
    const uint32_t sums_full_bar = bar_base + 8u * (2 * STAGES + 2 * L::kBuffers);       // the other CTAs' sums are here
    const uint32_t sums_taken_bar = bar_base + 8u * (2 * STAGES + 2 * L::kBuffers + 1);  // the others have read what this CTA sent
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t rank = ptx::cluster_cta_rank();
    const uint32_t cluster = blockIdx.x / S;
    const uint32_t num_clusters = gridDim.x / S;
    const uint32_t all_kb = (p.k + kF8BlockK - 1) / kF8BlockK;
    const uint32_t per_cta = (all_kb + S - 1) / S;
    const uint32_t kb0 = min(rank * per_cta, all_kb);
    const uint32_t num_kb = min(per_cta, all_kb - kb0);  // may be 0 in the last CTAs
    const uint32_t tiles = p.tiles_m * p.tiles_n;  // the blocks of A run fastest: they share a block of B
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_a);
        ptx::prefetch_tensormap(&tma_b);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (uint32_t b = 0; b < L::kBuffers; ++b) {
            ptx::mbar_init(acc_full_bar(b), 1);
            ptx::mbar_init(acc_empty_bar(b), L::kWarps);
        }
        ptx::mbar_init(sums_full_bar, (S - 1) * L::kWarps);
        ptx::mbar_init(sums_taken_bar, (S - 1) * L::kWarps);
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
        // The first blocks of B come to L2 while the kernel before (often the quantiser of A) ends: quantiser and product of 16 x
        // 16384 x 4096 together 16.9 -> 16.3 us, the product alone as before; twice and four times as far ahead, it lost.
        if (threadIdx.x == 32 && cluster < tiles)
            for (uint32_t kb = 0; kb < min(num_kb, STAGES); ++kb)
                ptx::tma_prefetch_2d(&tma_b, static_cast<int32_t>((kb0 + kb) * kF8BlockK),
                                     static_cast<int32_t>(cluster / p.tiles_m * f.bn));
        ptx::grid_dependency_wait();
    }

    bool role_ok = true;
    if (warp == 0) {
        // --------------------------------------------------- TMA producer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            const uint32_t bytes = (f.bn + REPL * min(p.m, kBlockM)) * kF8BlockK;
            for (uint32_t t = cluster; ok && t < tiles; t += num_clusters) {
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = wait_bounded(empty_bar(stage), phase ^ 1u, ctl, 1);
                    if (!ok)
                        break;
                    const uint32_t sa = smem_base + stage * L::kStageBytes;
                    const int32_t kx = static_cast<int32_t>((kb0 + kb) * kF8BlockK);
                    ptx::mbar_arrive_expect_tx(full_bar(stage), bytes);
                    ptx::tma_load_2d(sa + L::kABytes, &tma_b, full_bar(stage), kx, static_cast<int32_t>(t / p.tiles_m * f.bn));
#pragma unroll
                    for (uint32_t r = 0; r < REPL; ++r)
                        ptx::tma_load_2d(sa + r * L::kRows * kF8BlockK, &tma_a, full_bar(stage), kx,
                                         static_cast<int32_t>(t % p.tiles_m * kBlockM));
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
        // ---------------------------------------------------- MMA issuer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            uint32_t acc = 0, acc_phase = 0;
            bool ok = true;
            const uint32_t idesc = ptx::make_instr_desc_e4m3(kBlockM, f.bn);
            for (uint32_t t = cluster; ok && t < tiles; t += num_clusters) {
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = wait_bounded(full_bar(stage), phase, ctl, 2) &&
                         wait_bounded(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sa = smem_base + stage * L::kStageBytes;
                    const uint64_t da = ptx::make_smem_desc_sw128(sa);
                    const uint64_t db = ptx::make_smem_desc_sw128(sa + L::kABytes);
#pragma unroll
                    for (uint32_t k = 0; k < kF8BlockK / kF8UmmaK; ++k)
                        ptx::mma_f8_1cta(tmem_base + acc * L::kTileCols, da + 2u * k, db + 2u * k, idesc, k != 0u ? 1u : 0u);
                    ptx::mma_commit_1cta(acc_full_bar(acc));
                    ptx::mma_commit_1cta(empty_bar(stage));
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (++acc == L::kBuffers) {
                        acc = 0;
                        acc_phase ^= 1u;
                    }
                }
            }
            role_ok = ok;
        }
        __syncwarp();
    } else {
        // ---------------------------------------------- promotion and epilogue --
        const uint32_t quarter = warp & 3u, w = warp - 2u;
        // this warp's rows of A and columns of the tile
        const uint32_t warp_row = REPL == 4 ? 0u : (REPL == 2 ? (quarter & 1u) * 32u : quarter * 32u);
        const uint32_t col0 = (REPL == 4 ? quarter * 64u : (REPL == 2 ? (quarter >> 1) * 128u : 0u)) + (w >> 2) * L::kWarpCols;
        const uint32_t lane_addr = tmem_base + ((quarter * 32u) << 16) + col0;
        const uint32_t last_block = (p.n - 1) / 128u, last_kb = num_kb > 0 ? num_kb - 1 : 0u;
        const uint32_t exchange = smem_base + L::kExchangeOffset;
        uint32_t acc = 0, acc_phase = 0, parity = 0;
        bool ok = true;
        for (uint32_t t = cluster; ok && t < tiles; t += num_clusters, parity ^= 1u) {
            const uint32_t n0 = t / p.tiles_m * f.bn, row0 = t % p.tiles_m * kBlockM + warp_row;
            const float *sa = f.sa + static_cast<uint64_t>(min(row0 + lane, p.m - 1)) * f.ld_sa + kb0;
            // the (at most two) scale blocks of this warp's columns; bit c of `second`: chunk c lies in the second
            const uint32_t block0 = (n0 + col0) / 128u;
            uint32_t second = 0;
#pragma unroll
            for (uint32_t c = 0; c < kChunks; ++c)
                second |= (n0 + col0 + 32u * c) / 128u != block0 ? 1u << c : 0u;
            const float *sb0 = f.sb + static_cast<uint64_t>(min(block0, last_block)) * f.ld_sb + kb0;
            const float *sb1 = f.sb + static_cast<uint64_t>(min(block0 + 1u, last_block)) * f.ld_sb + kb0;
            const uint32_t cols = f.bn > col0 ? min(L::kWarpCols, f.bn - col0) : 0u;  // of this warp in the tile
            uint64_t sum[L::kWarpCols / 2];
#pragma unroll
            for (uint32_t i = 0; i < L::kWarpCols / 2; ++i)
                sum[i] = 0ull;
            float a0 = 0.0f, a1 = 0.0f, x0 = 0.0f, x1 = 0.0f, y0 = 0.0f, y1 = 0.0f;
            if (num_kb > 0) {  // the scales of the next two k-blocks are on their way behind this one's work
                const uint32_t one = min(1u, last_kb);
                a0 = ptx::ld_f32(sa), x0 = ptx::ld_f32(sb0), y0 = ptx::ld_f32(sb1);
                a1 = ptx::ld_f32(sa + one), x1 = ptx::ld_f32(sb0 + one), y1 = ptx::ld_f32(sb1 + one);
            }
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                const float s0 = a0 * x0, s1 = a0 * y0;
                const bool serve = f8_product_serves(a0, x0, s0) && f8_product_serves(a0, y0, s1);
                const uint32_t ahead = min(kb + 2, last_kb);
                a0 = a1, x0 = x1, y0 = y1;
                a1 = ptx::ld_f32(sa + ahead), x1 = ptx::ld_f32(sb0 + ahead), y1 = ptx::ld_f32(sb1 + ahead);
                ok = wait_bounded(acc_full_bar(acc), acc_phase, ctl, 3);
                const bool usual = __all_sync(0xffffffffu, ok && serve);  // one vote for both
                if (!usual) {
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok)
                        break;
                }
                ptx::tcgen05_fence_after();
                const uint32_t taddr = lane_addr + acc * L::kTileCols;
                auto promote = [&](uint32_t c, uint32_t(&v)[32]) {
                    const bool next = ((second >> c) & 1u) != 0u;
                    float s = next ? s1 : s0;
                    if (!usual)
                        s = f8_prescale(v, ptx::ld_f32(sa + kb), ptx::ld_f32((next ? sb1 : sb0) + kb));
                    f8_promote<L::kWarpCols / 2>(sum, 16 * c, v, ptx::pack_f32x2(__float_as_uint(s), __float_as_uint(s)));
                };
                uint32_t v0[32], v1[32];
                if (cols > 0) {
                    ptx::tmem_ld_32x32b_x32(taddr, v0);
                    if (kChunks == 2 && cols > 32)
                        ptx::tmem_ld_32x32b_x32(taddr + 32u, v1);
                    ptx::tmem_ld_wait();
                }
                // all columns are in registers: the buffer goes back
                ptx::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(acc_empty_bar(acc));
                if (cols > 0) {
                    promote(0, v0);
                    if constexpr (kChunks == 2)
                        if (cols > 32)
                            promote(1, v1);
                }
                if (++acc == L::kBuffers) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            if (!ok)
                break;
            // Every CTA finishes its share of each warp's columns: the others' sums of it come here, what this CTA has of theirs
            // goes there, once they have read what it sent for its tile before.
            ok = wait_bounded<true>(sums_taken_bar, parity ^ 1u, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
#pragma unroll
            for (uint32_t d = 0; d < S; ++d) {
                if (d == rank)
                    continue;
                // the slot of this CTA among the others of CTA d
                const uint32_t slot = rank - (rank > d ? 1u : 0u);
                const uint32_t to = ptx::mapa_shared(exchange + slot * L::kPartBytes + w * (L::kShare * 128u) + lane * 16u, d);
#pragma unroll
                for (uint32_t i = 0; i < L::kShare / 4; ++i) {
                    uint32_t q[4];
                    ptx::unpack_f32x2(sum[d * (L::kShare / 2) + 2 * i], q[0], q[1]);
                    ptx::unpack_f32x2(sum[d * (L::kShare / 2) + 2 * i + 1], q[2], q[3]);
                    ptx::st_shared_cluster_v4(to + i * 512u, q[0], q[1], q[2], q[3]);
                }
            }
            __syncwarp();
            // one lane per CTA: each release at cluster scope waits for what was stored, one after the other they would add up
            if (lane < S && lane != rank)
                ptx::mbar_arrive_cluster_addr(ptx::mapa_shared(sums_full_bar, lane));
            float mine[L::kShare];
#pragma unroll
            for (uint32_t d = 0; d < S; ++d)
                if (d == rank) {
#pragma unroll
                    for (uint32_t i = 0; i < L::kShare / 2; ++i) {
                        uint32_t lo, hi;
                        ptx::unpack_f32x2(sum[d * (L::kShare / 2) + i], lo, hi);
                        mine[2 * i] = __uint_as_float(lo), mine[2 * i + 1] = __uint_as_float(hi);
                    }
                }
            ok = wait_bounded<true>(sums_full_bar, parity, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            // in the order of the parts of K, whoever adds
            const uint8_t *from = smem_gen + L::kExchangeOffset + w * (L::kShare * 128u) + lane * 16u;
            uint32_t out[L::kShare];
#pragma unroll
            for (uint32_t i = 0; i < L::kShare / 4; ++i) {
                float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t d = 0; d < S; ++d) {
                    float4 part = make_float4(mine[4 * i], mine[4 * i + 1], mine[4 * i + 2], mine[4 * i + 3]);
                    if (d != rank)
                        part = *reinterpret_cast<const float4 *>(from + (d - (d > rank ? 1u : 0u)) * L::kPartBytes + i * 512u);
                    total.x += part.x, total.y += part.y, total.z += part.z, total.w += part.w;
                }
                out[4 * i] = __float_as_uint(total.x), out[4 * i + 1] = __float_as_uint(total.y);
                out[4 * i + 2] = __float_as_uint(total.z), out[4 * i + 3] = __float_as_uint(total.w);
            }
            __syncwarp();
            // ---- store this CTA's share: kShare columns of 32 rows (what came for this warp has been read: its place serves)
            const uint32_t end = min(p.n, n0 + f.bn), out_col = n0 + col0 + rank * L::kShare;
            if (row0 < p.m && out_col < end)
                store_share<L::kShare>(p, exchange + w * (L::kShare * 128u), lane, row0, out_col, end, out);
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
