// Products of e4m3 operands with a scale for each block of 128 along K:
//
//     C[m, n] = sum over k-blocks j of  sa[m, j] * sb[n / 128, j] * sum over k in block j of  qa[m, k] * qb[n, k]
//
// sa: one fp32 per row of A and k-block; sb: one fp32 per 128 x 128 block of B.  The inner sum is one tensor-core pass over
// 128 k (four tcgen05.mma.kind::f8f6f4 of 32), the outer one runs in fp32 registers ("promotion"): any scales, also where the
// product of the two is out of fp32's range (f8_prescale below), no rounding but fp32's until C is rounded to bf16 once.
//
// A CTA pair computes a 256 x 256 tile (128 x 256 per CTA).  One k-block of both operands is one 128-byte swizzle row, so
// the ring looks like the bf16 kernel's with twice the k per byte.  TMEM holds two accumulator buffers of 256 columns, one
// k-block each: while the MMA fills one, eight promotion warps read the other (`tcgen05.ld`), multiply by the two scales
// and add to 128 fp32 registers per thread; they hand the buffer back as soon as its last column is in registers.
//
// Bound: per k-block and SM the MMA needs 512 cycles, the TMEM read 256 (512 bytes a cycle), the fp32 multiply-adds 256
// issue slots per scheduler.  A block takes about 860 cycles: the two issuers (waits, four MMAs, two commits) and the promotion
// warps (wait, vote, scales, 330 cycles until the buffer goes back, the rest of the sums) are each that long, latencies and
// not pipes (FMA 40 % busy), and taking work out of one of them alone gains 3 % or less (three quarters of the scale loads: nothing; half
// the multiply-adds: 3 %).  8192^3: 478 to 558 us as the part's power allows (2.0 to 2.3 PFLOP/s).
#pragma once
#include "gemm_common.cuh"

namespace maize {

constexpr uint32_t kF8BlockK = 128;        // e4m3 elements per k-block = one 128-byte swizzle row = one scale
constexpr uint32_t kF8UmmaK = 32;          // K per tcgen05.mma for 8-bit operands
constexpr uint32_t kF8PromoteWarps = 8;    // two per quarter of the lanes: columns 0-127 and 128-255
constexpr uint32_t kF8ControlWarps = 4;    // producer, two MMA issuers, one idle: a whole warpgroup, so that it can give registers away
constexpr uint32_t kF8Threads = 32 * (kF8ControlWarps + kF8PromoteWarps);
// 384 threads are launched with 168 registers each (504 over the three warpgroups); the control warpgroup keeps 56, the two
// promotion warpgroups take 224 each: 56 + 2 * 224 = 504.
constexpr int kF8ControlRegs = 56;
constexpr int kF8PromoteRegs = 224;

struct F8Params {
    GemmParams g;
    const float *sa, *sb;
    uint64_t ld_sa, ld_sb;  // row pitches of the scales
};

// Two staging buffers of 32 rows x 64 columns for each promotion warp: both stores of a tile are on their way before the warp
// goes on (with one, and a sixth ring stage: 8192 x 8192 x 512 54 us instead of 50, 4096 x 4096 x 1024 25.4 instead of 24.2).
constexpr uint32_t kF8StageWarpBytes = 2 * kTmaStoreBufBytes;

template <uint32_t STAGES>
struct F8SmemLayout {
    static constexpr uint32_t kABytes = kBlockM * kF8BlockK;
    static constexpr uint32_t kBBytes = 128 * kF8BlockK;  // this CTA's half of the 256 columns
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr uint32_t kStagingOffset = STAGES * kStageBytes;
    static constexpr uint32_t kStagingBytes = kF8PromoteWarps * kF8StageWarpBytes;
    static constexpr uint32_t kBarOffset = kStagingOffset + kStagingBytes;
    static constexpr uint32_t kNumBars = 2 * STAGES + 6;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kUsedBytes = kAbortOffset + 4;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
};

// Stores 32 rows x 64 columns of C that lie in `stage` as 128-byte rows, 16-byte chunk j of row r at chunk j ^ (r & 7), to
// rows of any alignment: a lane stores 4 bytes, so a row leaves as one run of 128.  Where a row starts between two words
// the lanes pass on a half, and the ends of the run are 2-byte stores.  (2-byte stores throughout: 4111 x 3967 x 4112 in 125 us
// instead of 81; with rows for TMA 75.)
__device__ __forceinline__ void f8_store_rows(const GemmParams &p, uint32_t stage_u32, uint32_t lane, uint32_t row0, uint32_t col0)
{
    const uint32_t rows = min(32u, p.m - row0);
    const uint32_t left = p.n - col0;  // columns there are
    const uint32_t chunk = lane >> 2, word = (lane & 3u) * 4u;
    __nv_bfloat16 *dst = p.c + static_cast<uint64_t>(row0) * p.ldc + col0;
    if (rows == 32u && left >= 64u) {
        // every row the same way, but for whether it starts between two words: with an odd pitch every other one does
        const bool first = (reinterpret_cast<uintptr_t>(dst) & 2u) != 0u, odd_pitch = (p.ldc & 1u) != 0u;
        __nv_bfloat16 *to = dst + 2u * lane;
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < 32; r0 += 16) {
            uint32_t v[16];
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i)
                v[i] = ptx::ld_shared_u32(stage_u32 + (r0 + i) * 128u + ((chunk ^ (i & 7u)) << 4) + word);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                if (first != (odd_pitch && (i & 1u) != 0u)) {
                    const uint32_t before = __shfl_up_sync(0xffffffffu, v[i], 1);
                    if (lane != 0u)
                        *reinterpret_cast<uint32_t *>(to - 1) = __funnelshift_l(before, v[i], 16);
                } else {
                    *reinterpret_cast<uint32_t *>(to) = v[i];
                }
                to += p.ldc;
            }
        }
        // the first and the last column of the rows that start between words: a lane for each of 32 such ends
        if (first || odd_pitch) {
            for (uint32_t pass = 0; pass < (odd_pitch ? 1u : 2u); ++pass) {
                const uint32_t r = odd_pitch ? (lane >> 1) * 2u + (first ? 0u : 1u) : pass * 16u + (lane >> 1);
                const uint32_t c = (lane & 1u) * 63u;
                dst[static_cast<uint64_t>(r) * p.ldc + c] =
                    ptx::ld_shared_bf16(stage_u32 + r * 128u + (((c >> 3) ^ (r & 7u)) << 4) + (c & 7u) * 2u);
            }
        }
        __syncwarp();
        return;
    }
#pragma unroll 1
    for (uint32_t r = 0; r < rows; ++r) {
        // at the edges of C: two columns per lane, each by itself
        const uint32_t mine = ptx::ld_shared_u32(stage_u32 + r * 128u + ((chunk ^ (r & 7u)) << 4) + word);
        if (2u * lane < left)
            *reinterpret_cast<uint16_t *>(dst + 2u * lane) = static_cast<uint16_t>(mine);
        if (2u * lane + 1u < left)
            *reinterpret_cast<uint16_t *>(dst + 2u * lane + 1u) = static_cast<uint16_t>(mine >> 16);
        dst += p.ldc;
    }
    __syncwarp();
}

// Writes this warp's 32 rows x 128 columns of C, held as 128 fp32 per lane (lane = row): through the warp's staging buffers
// and TMA stores, or f8_store_rows where C's rows are not for TMA.  A buffer for each half.  At the right edge of C a tile may
// have the first half only, so how many stores lie between two of one buffer is not known: before the first half all of the
// tile before have read theirs.  They had this tile's sum to do it in (buffers that alternate with every store and a wait for
// all but the last one: 8192^3 553 us instead of 536).
__device__ __forceinline__ void f8_store(const GemmParams &p, const CUtensorMap *tma_c, uint32_t stage_u32, uint32_t lane,
                                         uint32_t row0, uint32_t col0, const uint64_t (&acc)[64])
{
    if (row0 >= p.m)
        return;
#pragma unroll
    for (uint32_t g = 0; g < 2; ++g) {
        const uint32_t col = col0 + g * 64u;
        if (col < p.n) {
            if (g == 0) {
                if (p.c_tma_ok && lane == 0)
                    ptx::bulk_wait_group_read<0>();
                __syncwarp();
            }
            const uint32_t buffer = stage_u32 + g * kTmaStoreBufBytes;
            const uint32_t row = buffer + lane * 128u;
            const uint32_t sw = lane & 7u;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                uint32_t w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t lo, hi;
                    ptx::unpack_f32x2(acc[g * 32 + 4 * j + i], lo, hi);
                    w[i] = ptx::pack_bf16x2(lo, hi);
                }
                ptx::st_shared_v4(row + ((j ^ sw) << 4), w[0], w[1], w[2], w[3]);
            }
            if (p.c_tma_ok) {
                ptx::fence_proxy_async_shared();
                __syncwarp();
                if (lane == 0) {
                    ptx::tma_store_2d(tma_c, buffer, static_cast<int32_t>(col), static_cast<int32_t>(row0));
                    ptx::bulk_commit_group();
                }
            } else {
                __syncwarp();
                f8_store_rows(p, buffer, lane, row0, col);
            }
        }
    }
}

// acc[first .. first + 15] += v * ss: 32 columns of one row, in pairs.
template <uint32_t PAIRS>
__device__ __forceinline__ void f8_promote(uint64_t (&acc)[PAIRS], int first, const uint32_t (&v)[32], uint64_t ss)
{
#pragma unroll
    for (int i = 0; i < 16; ++i)
        ptx::fma_f32x2(acc[first + i], ptx::pack_f32x2(v[2 * i], v[2 * i + 1]), ss);
}

// The sums of a block are multiplied by the product of its two scales where that is a normal number or one of them is zero.  A
// product that overflows, or loses bits below 2^-126, says nothing about the sums times both.
__device__ __forceinline__ bool f8_product_serves(float a, float b, float product)
{
    return (fabsf(product) >= 1.17549435e-38f && fabsf(product) <= 3.40282347e38f) || a == 0.0f || b == 0.0f;
}

// Where it does not serve: v *= the larger scale, and the answer is the smaller one, for f8_promote.  In this order nothing goes
// out of range that the result does not.  Lanes whose product serves keep v and get the product, so that a row's result does
// not depend on its neighbours' scales.
__device__ __forceinline__ float f8_prescale(uint32_t (&v)[32], float a, float b)
{
    const float product = a * b;
    const bool serves = f8_product_serves(a, b, product), a_first = fabsf(a) > fabsf(b);
    const float larger = serves ? 1.0f : (a_first ? a : b);
#pragma unroll
    for (int i = 0; i < 32; ++i)
        v[i] = __float_as_uint(__uint_as_float(v[i]) * larger);
    return serves ? product : (a_first ? b : a);
}

template <uint32_t STAGES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kF8Threads, 1)
gemm_e4m3_sm100_2cta(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                     const __grid_constant__ CUtensorMap tma_c, const F8Params f)
{
    using L = F8SmemLayout<STAGES>;
    constexpr uint32_t kTmemCols = 512;
    constexpr uint32_t kIdesc = ptx::make_instr_desc_e4m3(2 * kBlockM, 256);
    const GemmParams &p = f.g;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    auto turn_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 4 + b); };  // the other issuer's MMAs are in the pipe
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t cta_rank = ptx::cluster_cta_rank();
    const uint32_t pair = blockIdx.x >> 1;
    const uint32_t num_pairs = gridDim.x >> 1;
    const uint32_t num_tiles = p.tiles_m * p.tiles_n;
    const uint32_t num_kb = (p.k + kF8BlockK - 1) / kF8BlockK;
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_a);
        ptx::prefetch_tensormap(&tma_b);
        if (p.c_tma_ok)
            ptx::prefetch_tensormap(&tma_c);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            ptx::mbar_init(acc_full_bar(b), 1);
            ptx::mbar_init(acc_empty_bar(b), 2 * kF8PromoteWarps);  // one lane per promotion warp of both CTAs
            ptx::mbar_init(turn_bar(b), 1);
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

    // Waits acquire at CTA scope: tensor memory and asynchronous copies come with the barrier's own phase, no thread's stores
    // do (with cluster scope 4111 x 3967 x 4112 took 81.6 us instead of 77.3, 4096 x 4096 x 7168 110 instead of 108).
    bool role_ok = true;
    if (warp < kF8ControlWarps) {
        ptx::setmaxnreg_dec<kF8ControlRegs>();
        if (warp == 0) {
            // ------------------------------------------------------- TMA producer --
            if (lane == 0) {
                uint32_t stage = 0, phase = 0;
                bool ok = true;
                for (uint32_t t = pair; ok && t < num_tiles; t += num_pairs) {
                    const TileCoord tc = tile_coord(t, p);
                    const int32_t m0 = static_cast<int32_t>(tc.m_blk * 2 * kBlockM + cta_rank * kBlockM);
                    const int32_t n0 = static_cast<int32_t>(tc.n_blk * 256u + cta_rank * 128u);
                    for (uint32_t kb = 0; kb < num_kb; ++kb) {
                        ok = wait_bounded(empty_bar(stage), phase ^ 1u, ctl, 1);
                        if (!ok)
                            break;
                        const uint32_t sa = smem_base + stage * L::kStageBytes;
                        const uint32_t leader_full = ptx::mapa_shared(full_bar(stage), 0);
                        if (cta_rank == 0)
                            ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * L::kStageBytes);
                        const int32_t kx = static_cast<int32_t>(kb * kF8BlockK);
                        ptx::tma_load_2d_pair(sa, &tma_a, leader_full, kx, m0);
                        ptx::tma_load_2d_pair(sa + L::kABytes, &tma_b, leader_full, kx, n0);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                role_ok = ok;
            }
            __syncwarp();
        } else if (warp == 1 || warp == 2) {
            // ------------------------------- MMA issuers (leader only), a buffer each --
            // Blocks of 128 k do not depend on each other: warp 1 issues the even ones, warp 2 the odd ones, and one does its waits and
            // commits (some 300 cycles a block) while the other's MMAs run (4096^3: 69 -> 66 us, 8192^3: 509 -> 489).  They take
            // turns: side by side in the pipe two blocks would both end late.
            if (lane == 0 && cta_rank == 0) {
                const uint32_t acc = warp - 1u;
                const uint32_t blocks = pair < num_tiles ? ((num_tiles - pair - 1u) / num_pairs + 1u) * num_kb : 0u;
                uint32_t stage = acc, phase = 0, acc_phase = 0;
                bool ok = true;
                for (uint32_t it = acc; it < blocks; it += 2) {
                    ok = wait_bounded(full_bar(stage), phase, ctl, 2) &&
                         wait_bounded(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2) &&
                         wait_bounded(turn_bar(acc), acc == 0u ? acc_phase ^ 1u : acc_phase, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sa = smem_base + stage * L::kStageBytes;
                    const uint64_t da = ptx::make_smem_desc_sw128(sa);
                    const uint64_t db = ptx::make_smem_desc_sw128(sa + L::kABytes);
                    const uint32_t tmem_d = tmem_base + acc * 256u;
    #pragma unroll
                    for (uint32_t k = 0; k < kF8BlockK / kF8UmmaK; ++k)
                        ptx::mma_f8_2cta(tmem_d, da + 2u * k, db + 2u * k, kIdesc, k != 0u ? 1u : 0u);
                    ptx::mbar_arrive(turn_bar(acc ^ 1u));
                    ptx::mma_commit_2cta_mask(acc_full_bar(acc), 3);
                    ptx::mma_commit_2cta_mask(empty_bar(stage), 3);
                    stage += 2;
                    if (stage >= STAGES) {
                        stage -= STAGES;
                        phase ^= 1u;
                    }
                    acc_phase ^= 1u;
                }
                role_ok = ok;
            }
            __syncwarp();
        }
    } else {
        ptx::setmaxnreg_inc<kF8PromoteRegs>();
        // ---------------------------------------------- promotion and epilogue --
        const uint32_t quarter = warp & 3u;
        const uint32_t half = (warp - kF8ControlWarps) >> 2;
        const uint32_t stage_u32 = smem_base + L::kStagingOffset + (warp - kF8ControlWarps) * kF8StageWarpBytes;
        const uint32_t lane_cols = tmem_base + ((quarter * 32u) << 16) + half * 128u;
        const uint32_t leader_empty0 = ptx::mapa_shared(acc_empty_bar(0), 0);
        uint32_t buf = 0, buf_phase = 0;
        bool ok = true;
        for (uint32_t t = pair; ok && t < num_tiles; t += num_pairs) {
            const TileCoord tc = tile_coord(t, p);
            const uint32_t row0 = tc.m_blk * 2 * kBlockM + cta_rank * kBlockM + quarter * 32u;
            const uint32_t col0 = tc.n_blk * 256u + half * 128u;
            const bool row_in = row0 + lane < p.m, col_in = col0 < p.n;
            const float *sa = f.sa + static_cast<uint64_t>(row_in ? row0 + lane : 0u) * f.ld_sa;
            const float *sb = f.sb + static_cast<uint64_t>(col_in ? col0 / 128u : 0u) * f.ld_sb;
            uint64_t acc[64];  // 128 fp32 in pairs of neighbouring columns
#pragma unroll
            for (int i = 0; i < 64; ++i)
                acc[i] = 0ull;
            // the scales of the next two k-blocks are on their way behind this one's work
            float a0 = ptx::ld_f32(sa), b0 = ptx::ld_f32(sb);
            const uint32_t last = num_kb - 1;
            float a1 = ptx::ld_f32(sa + min(1u, last)), b1 = ptx::ld_f32(sb + min(1u, last));
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                const float s = a0 * b0;
                const bool serves = f8_product_serves(a0, b0, s);
                a0 = a1, b0 = b1;
                a1 = ptx::ld_f32(sa + min(kb + 2, last));
                b1 = ptx::ld_f32(sb + min(kb + 2, last));
                ok = wait_bounded(acc_full_bar(buf), buf_phase, ctl, 3);
                const uint32_t taddr = lane_cols + buf * 256u;
                // Two loads of 32 columns in flight at a time: a load's latency, not its transfer, is what a warp waits for,
                // and tcgen05.wait::ld waits for all of them.
                uint32_t v0[32], v1[32];
                uint64_t ss = ptx::pack_f32x2(__float_as_uint(s), __float_as_uint(s));
                // For scales whose product is out of range.  They are loaded again, so that the usual block holds nothing for them, and the
                // usual block's first loads stand by themselves, so that it has one branch more than without (8192^3 541 us
                // instead of 533; two more 545; a second way through the whole block spills and takes up to twice as long).
                auto prescale = [&] {
                    const float a = ptx::ld_f32(sa + kb), b = ptx::ld_f32(sb + kb);
                    const uint32_t rest = __float_as_uint(f8_prescale(v0, a, b));
                    f8_prescale(v1, a, b);
                    ss = ptx::pack_f32x2(rest, rest);
                };
                const bool usual = __all_sync(0xffffffffu, ok && serves);  // one vote for both
                if (usual) {
                    ptx::tcgen05_fence_after();
                    ptx::tmem_ld_32x32b_x32(taddr, v0);
                    ptx::tmem_ld_32x32b_x32(taddr + 32u, v1);
                    ptx::tmem_ld_wait();
                } else {
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    ptx::tmem_ld_32x32b_x32(taddr, v0);
                    ptx::tmem_ld_32x32b_x32(taddr + 32u, v1);
                    ptx::tmem_ld_wait();
                    prescale();
                }
                f8_promote(acc, 0, v0, ss);
                ptx::tmem_ld_32x32b_x32(taddr + 64u, v0);
                f8_promote(acc, 16, v1, ss);
                ptx::tmem_ld_32x32b_x32(taddr + 96u, v1);
                ptx::tmem_ld_wait();
                // all columns are in registers: the buffer goes back
                ptx::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive_cluster_addr_relaxed(leader_empty0 + 8u * buf);
                if (!usual)
                    prescale();
                f8_promote(acc, 32, v0, ss);
                f8_promote(acc, 48, v1, ss);
                if (++buf == 2) {
                    buf = 0;
                    buf_phase ^= 1u;
                }
            }
            if (!ok)
                break;
            f8_store(p, &tma_c, stage_u32, lane, row0, col0, acc);
            __syncwarp();
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
