// The e4m3 product for few rows of A (M <= 128): bound by reading B once.
//
// As in the grouped product, B is the M side of the MMA (up to 128 of its rows per tile) and the rows of A its N side
// (NT = 16, 32, 64 or 128).  A cluster of two CTAs shares a tile and splits K: each takes half of the k-blocks, promotes
// them in registers (lane = row of B, one register per row of A) and sends the other CTA half of its sums through
// distributed shared memory; each then rounds and stores half of the rows of A.  No global scratch, a fixed order of sums.
//
// The tile's height is chosen by the host so that the tiles fill whole rounds of CTA pairs (16384 rows over 74 pairs: two
// rounds of 112 rows); a tile may then touch two scale blocks of B, so the scale of B is per lane.  The scales of A for this
// CTA's k-blocks are read once into shared memory, transposed.
//
// NT columns of TMEM per k-block leave room for four accumulator buffers, so the MMA never waits for a hand-over; the ring
// holds 6 to 10 stages of 128 k (128 bytes per row).
#pragma once
#include "gemm_e4m3_sm100.cuh"
#include "gemm_sm100_grouped.cuh"

namespace maize {

constexpr uint32_t kF8SkinnyMaxKb = 64;  // k-blocks per CTA whose scales fit in shared memory: K <= 16384

struct F8SkinnyParams {
    GroupedParams c;   // C, its pitch and alignment, n = N, k = K, rows = M (no offsets)
    const float *sa, *sb;
    uint64_t ld_sa, ld_sb;
    uint32_t tile_rows;  // rows of B per tile, a multiple of 8, at most 128
    uint32_t tiles;
};

template <uint32_t NT, uint32_t STAGES>
struct F8SkinnySmemLayout {
    static constexpr uint32_t kBBytes = 128 * kF8BlockK;
    static constexpr uint32_t kABytes = NT * kF8BlockK;
    static constexpr uint32_t kStageBytes = kBBytes + kABytes;
    static constexpr uint32_t kExchangeOffset = STAGES * kStageBytes;  // the other CTA's sums for this CTA's half of the rows
    static constexpr uint32_t kExchangeBytes = 128 * (NT / 2) * 4;
    static constexpr uint32_t kScaleAOffset = kExchangeOffset + kExchangeBytes;
    static constexpr uint32_t kScaleABytes = kF8SkinnyMaxKb * NT * 4;
    static constexpr uint32_t kScaleBOffset = kScaleAOffset + kScaleABytes;  // two scale blocks x k-blocks, for two tiles
    static constexpr uint32_t kScaleBBytes = 2 * 2 * kF8SkinnyMaxKb * 4;
    static constexpr uint32_t kBarOffset = kScaleBOffset + kScaleBBytes;
    static constexpr uint32_t kNumBars = 2 * STAGES + 8 + 2;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kUsedBytes = kAbortOffset + 4;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
};

// sum[i] += v[i] * (scale of row i of A * scale of this lane's row of B)
template <int N>
__device__ __forceinline__ void f8_skinny_promote(float *sum, const uint32_t (&v)[N], const float4 *sa, float sb)
{
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 s = sa[i];
        sum[4 * i + 0] = fmaf(__uint_as_float(v[4 * i + 0]), s.x * sb, sum[4 * i + 0]);
        sum[4 * i + 1] = fmaf(__uint_as_float(v[4 * i + 1]), s.y * sb, sum[4 * i + 1]);
        sum[4 * i + 2] = fmaf(__uint_as_float(v[4 * i + 2]), s.z * sb, sum[4 * i + 2]);
        sum[4 * i + 3] = fmaf(__uint_as_float(v[4 * i + 3]), s.w * sb, sum[4 * i + 3]);
    }
}

template <uint32_t NT, uint32_t STAGES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNumThreads, 1)
gemm_e4m3_sm100_skinny(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                       const F8SkinnyParams f)
{
    using L = F8SkinnySmemLayout<NT, STAGES>;
    static_assert(NT == 16 || NT == 32 || NT == 64 || NT == 128, "rows of A per launch");
    constexpr uint32_t kBuffers = 4;
    constexpr uint32_t kTmemCols = kBuffers * NT;  // 64 .. 512
    constexpr uint32_t kIdesc = ptx::make_instr_desc_e4m3(kBlockM, NT);
    constexpr uint32_t kHalf = NT / 2;
    const GroupedParams &p = f.c;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + kBuffers + b); };
    const uint32_t sums_full_bar = bar_base + 8u * (2 * STAGES + 2 * kBuffers);        // the peer's sums are here
    const uint32_t sums_taken_bar = bar_base + 8u * (2 * STAGES + 2 * kBuffers + 1);   // the peer has read what this CTA sent
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t cta_rank = ptx::cluster_cta_rank();
    const uint32_t pair = blockIdx.x >> 1;
    const uint32_t num_pairs = gridDim.x >> 1;
    const uint32_t all_kb = (p.k + kF8BlockK - 1) / kF8BlockK;
    const uint32_t first_half = (all_kb + 1) / 2;
    const uint32_t kb0 = cta_rank == 0 ? 0u : first_half;
    const uint32_t num_kb = cta_rank == 0 ? first_half : all_kb - first_half;  // 0 in the second CTA if K is one block
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_a);
        ptx::prefetch_tensormap(&tma_b);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (uint32_t b = 0; b < kBuffers; ++b) {
            ptx::mbar_init(acc_full_bar(b), 1);
            ptx::mbar_init(acc_empty_bar(b), kNumEpilogueWarps);
        }
        ptx::mbar_init(sums_full_bar, kNumEpilogueWarps);
        ptx::mbar_init(sums_taken_bar, kNumEpilogueWarps);
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

    bool role_ok = true;
    if (warp == 0) {
        // ------------------------------------------------------- TMA producer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            const uint32_t bytes = f.tile_rows * kF8BlockK + L::kABytes;
            for (uint32_t t = pair; ok && t < f.tiles; t += num_pairs) {
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = wait_bounded(empty_bar(stage), phase ^ 1u, ctl, 1);
                    if (!ok)
                        break;
                    const uint32_t sb = smem_base + stage * L::kStageBytes;
                    const int32_t kx = static_cast<int32_t>((kb0 + kb) * kF8BlockK);
                    ptx::mbar_arrive_expect_tx(full_bar(stage), bytes);
                    ptx::tma_load_2d(sb, &tma_b, full_bar(stage), kx, static_cast<int32_t>(t * f.tile_rows));
                    ptx::tma_load_2d(sb + L::kBBytes, &tma_a, full_bar(stage), kx, 0);
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
            for (uint32_t t = pair; ok && t < f.tiles; t += num_pairs) {
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    ok = wait_bounded(full_bar(stage), phase, ctl, 2) &&
                         wait_bounded(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sb = smem_base + stage * L::kStageBytes;
                    const uint64_t db = ptx::make_smem_desc_sw128(sb);
                    const uint64_t da = ptx::make_smem_desc_sw128(sb + L::kBBytes);
#pragma unroll
                    for (uint32_t k = 0; k < kF8BlockK / kF8UmmaK; ++k)
                        ptx::mma_f8_1cta(tmem_base + acc * NT, db + 2u * k, da + 2u * k, kIdesc, k != 0u ? 1u : 0u);
                    ptx::mma_commit_1cta(acc_full_bar(acc));
                    ptx::mma_commit_1cta(empty_bar(stage));
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (++acc == kBuffers) {
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
        const uint32_t quarter = warp & 3u;
        const uint32_t row = quarter * 32u + lane;  // of the tile's rows of B
        const uint32_t tid = threadIdx.x - 64u;     // 0 .. 127
        float *scale_a = reinterpret_cast<float *>(smem_gen + L::kScaleAOffset);  // [k-block][row of A]
        float *scale_b = reinterpret_cast<float *>(smem_gen + L::kScaleBOffset);  // [tile parity][scale block][k-block]
        float *sums_in = reinterpret_cast<float *>(smem_gen + L::kExchangeOffset);  // [row of A][128]
        const uint32_t sums_out = ptx::mapa_shared(smem_base + L::kExchangeOffset, cta_rank ^ 1u);
        const uint32_t peer_full = ptx::mapa_shared(sums_full_bar, cta_rank ^ 1u);
        const uint32_t peer_taken = ptx::mapa_shared(sums_taken_bar, cta_rank ^ 1u);
        const uint32_t last_block = (p.n - 1) / 128u;
        // thread i < 2 * 64 fetches scale block i / 64, k-block i % 64 of a tile
        auto fetch_scale_b = [&](uint32_t t) {
            const uint32_t kb = tid & (kF8SkinnyMaxKb - 1);
            const uint32_t block = min(t * f.tile_rows / 128u + tid / kF8SkinnyMaxKb, last_block);
            return t < f.tiles && kb < num_kb ? __ldg(f.sb + static_cast<uint64_t>(block) * f.ld_sb + kb0 + kb) : 0.0f;
        };
        float next_b = fetch_scale_b(pair);
        // eight loads in flight per thread: one after the other they cost 16 latencies for 128 rows and 16 k-blocks
        for (uint32_t base = tid; base < num_kb * NT; base += 8u * 128u) {
            float v[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint32_t i = base + u * 128u, m = i / num_kb, kb = i - m * num_kb;
                v[u] = m < p.rows && i < num_kb * NT ? __ldg(f.sa + static_cast<uint64_t>(m) * f.ld_sa + kb0 + kb) : 0.0f;
            }
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint32_t i = base + u * 128u, m = i / num_kb, kb = i - m * num_kb;
                if (i < num_kb * NT)
                    scale_a[kb * NT + m] = v[u];
            }
        }
        uint32_t acc = 0, acc_phase = 0, parity = 0;
        bool ok = true;
        for (uint32_t t = pair; ok && t < f.tiles; t += num_pairs, parity ^= 1u) {
            const uint32_t n0 = t * f.tile_rows;
            float *my_b = scale_b + parity * 2 * kF8SkinnyMaxKb;
            my_b[tid] = next_b;
            asm volatile("bar.sync 1, 128;" ::: "memory");  // the scales of this tile (and of A) are in place
            next_b = fetch_scale_b(t + num_pairs);
            const float *lane_b = my_b + ((n0 + row) / 128u - n0 / 128u) * kF8SkinnyMaxKb;
            float sum[NT];
#pragma unroll
            for (uint32_t i = 0; i < NT; ++i)
                sum[i] = 0.0f;
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                ok = wait_bounded(acc_full_bar(acc), acc_phase, ctl, 3);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t taddr = tmem_base + acc * NT + ((quarter * 32u) << 16);
                const float sb = lane_b[kb];
                const float4 *sa = reinterpret_cast<const float4 *>(scale_a + kb * NT);
                auto hand_back = [&]() {
                    ptx::tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        ptx::mbar_arrive(acc_empty_bar(acc));
                };
                if constexpr (NT == 16) {
                    uint32_t v[16];
                    ptx::tmem_ld_32x32b_x16(taddr, v);
                    ptx::tmem_ld_wait();
                    hand_back();
                    f8_skinny_promote(sum, v, sa, sb);
                } else {
                    // at most two loads of 32 columns in flight, the buffer back as soon as the last is in registers
                    uint32_t v0[32], v1[32];
                    ptx::tmem_ld_32x32b_x32(taddr, v0);
                    if constexpr (NT >= 64)
                        ptx::tmem_ld_32x32b_x32(taddr + 32u, v1);
                    ptx::tmem_ld_wait();
                    if constexpr (NT == 128) {
                        f8_skinny_promote(sum, v0, sa, sb);
                        ptx::tmem_ld_32x32b_x32(taddr + 64u, v0);
                        f8_skinny_promote(sum + 32, v1, sa + 8, sb);
                        ptx::tmem_ld_32x32b_x32(taddr + 96u, v1);
                        ptx::tmem_ld_wait();
                    }
                    hand_back();
                    constexpr uint32_t kDone = NT == 128 ? 64u : 0u;
                    f8_skinny_promote(sum + kDone, v0, sa + kDone / 4, sb);
                    if constexpr (NT >= 64)
                        f8_skinny_promote(sum + kDone + 32, v1, sa + kDone / 4 + 8, sb);
                }
                if (++acc == kBuffers) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            if (!ok)
                break;
            // The sums of the other CTA's half of the rows of A go there; the exchange buffer has been read since the last tile.
            ok = wait_bounded<true>(sums_taken_bar, parity ^ 1u, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
#pragma unroll
            for (uint32_t i = 0; i < kHalf; ++i)
                ptx::st_shared_cluster_u32(sums_out + (i * 128u + row) * 4u,
                                           __float_as_uint(cta_rank == 0 ? sum[kHalf + i] : sum[i]));
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive_cluster_addr(peer_full);
            ok = wait_bounded<true>(sums_full_bar, parity, ctl, 7);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            uint32_t out[kHalf < 32 ? 32 : kHalf] = {};
#pragma unroll
            for (uint32_t i = 0; i < kHalf; ++i) {
                const float mine = cta_rank == 0 ? sum[i] : sum[kHalf + i], theirs = sums_in[i * 128u + row];
                // k order: the first CTA's blocks come first
                out[i] = __float_as_uint(cta_rank == 0 ? mine + theirs : theirs + mine);
            }
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive_cluster_addr(peer_taken);
            GroupedParams q = p;
            q.n = min(p.n, n0 + f.tile_rows);
            const uint32_t m0 = cta_rank * kHalf;
#pragma unroll
            for (uint32_t c = 0; c < kHalf; c += 32) {
                if (m0 + c < p.rows && n0 + quarter * 32u < q.n) {
                    uint32_t v[32];
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i)
                        v[i] = out[c + i];
                    store_transposed_chunk(q, m0 + c, min(min(32u, kHalf), p.rows - m0 - c), n0 + row, lane, v);
                }
                __syncwarp();
            }
        }
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
        ptx::tmem_dealloc_1cta(tmem_base, kTmemCols);
    }
}

}  // namespace maize
