// C ABI of the 8-bit products and their quantiser (declared in include/maize_gemm.h).
#include "../../include/maize_gemm.h"

#include <cstring>

#include "maize_host.cuh"
#include "gemm_e4m3_sm100.cuh"
#include "gemm_e4m3_sm100_skinny.cuh"
#include "quantize_e4m3.cuh"

namespace {

using maize::aligned;
using maize::DeviceGuard;
using maize::fail;
using maize::fail_cuda;

maize_status_t byte_map(maize_ctx_t *ctx, CUtensorMap *map, const void *base, uint64_t rows, uint64_t cols, uint64_t ld,
                        uint32_t box_rows)
{
    const uint64_t dims[2] = {cols, rows}, strides[1] = {ld};
    const uint32_t box[2] = {maize::kF8BlockK, box_rows};
    return maize::encode_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, 2, dims, strides, box,
                             static_cast<CUtensorMapL2promotion>(ctx->tma_promotion));
}

template <uint32_t REPL, uint32_t S, uint32_t STAGES>
maize_status_t launch_skinny(maize_ctx_t *ctx, int slot, uint32_t clusters, const CUtensorMap &ta, const CUtensorMap &tb,
                             const maize::F8SkinnyParams &f, cudaStream_t stream)
{
    using L = maize::F8SkinnyLayout<REPL, S, STAGES>;
    const uint64_t tiles = uint64_t(f.g.tiles_m) * f.g.tiles_n;
    const uint32_t grid = (tiles < clusters ? static_cast<uint32_t>(tiles) : clusters) * S;
    return maize::launch_clusters(ctx, slot, maize::gemm_e4m3_sm100_skinny<REPL, S, STAGES>, grid, S, maize::kF8SkinnyThreads,
                                  L::kDynamicBytes, stream, ta, tb, f);
}

// How the tiles of a product with K split over clusters are cut.
struct SkinnyPlan {
    uint32_t copies;    // of the rows of A in an MMA's 128 lanes
    uint32_t parts;     // CTAs that share a tile's K
    uint32_t clusters;  // at a time
    uint32_t tiles_m;   // blocks of 128 rows of A
    uint32_t bn;        // rows of B per tile
    double cost;        // microseconds beyond what every call takes, for comparison only
};

// The tiles are as wide as fills whole rounds of clusters.  A k-block costs a CTA 0.34 us (the MMA thread's issue and the
// hand-over of its accumulator) or its bytes at 80 GB/s per SM (47 with 128 different rows of A), a tile's end 2 to 3.5 us by the
// rows there are (rounds of 50000 x 512: 3 us each for 16 rows, 5.1 for 33, 4.6 for 65), measured; joining four parts about 0.8
// us more than joining two.  16 x 512 x 8192: 9.8 us in four parts, 14.7 in two; 5 x 9001 x 2048: 12.8, 7.8.
SkinnyPlan skinny_plan(maize_ctx_t *ctx, uint32_t parts, uint32_t m, uint32_t n, uint32_t kblocks)
{
    SkinnyPlan q;
    q.copies = m <= 32 ? 4 : (m <= 64 ? 2 : 1);
    q.parts = parts;
    q.tiles_m = (m + 127) / 128;
    q.clusters = maize::clusters_at_once(ctx, parts, maize::gemm_e4m3_sm100_skinny<1, 4, 5>, maize::kF8SkinnyThreads,
                                         maize::F8SkinnyLayout<1, 4, 5>::kDynamicBytes);
    const uint64_t widest = q.copies == 1 ? 128 : 256;
    const uint64_t rounds = (uint64_t(q.tiles_m) * ((n + widest - 1) / widest) + q.clusters - 1) / q.clusters;
    uint64_t per_m = rounds * q.clusters / q.tiles_m;  // tiles along N that fill the rounds
    if (per_m == 0)
        per_m = 1;
    uint64_t bn = ((n + per_m - 1) / per_m + 31) / 32 * 32;
    q.bn = static_cast<uint32_t>(bn < widest ? bn : widest);
    const double bytes = (q.bn + q.copies * (m < 128 ? m : 128u)) * 128.0;
    const double rate = q.copies == 1 ? 47e3 : 80e3, block = bytes / rate > 0.34 ? bytes / rate : 0.34;
    const double end = (q.copies == 4 ? 2.0 : (q.copies == 2 ? 3.5 : 3.2)) + (parts == 2 ? 0.0 : 0.8);
    q.cost = double(rounds) * (((kblocks + parts - 1) / parts) * block + end);
    return q;
}

maize_status_t skinny(maize_ctx_t *ctx, const SkinnyPlan &plan, const void *a, uint64_t lda, const float *sa, uint64_t ld_sa,
                      const void *b, uint64_t ldb, const float *sb, uint64_t ld_sb, void *c, uint64_t ldc, uint32_t m, uint32_t n,
                      uint32_t k, cudaStream_t stream)
{
    const uint32_t bn = plan.bn;
    if (uint64_t(plan.tiles_m) * ((uint64_t(n) + bn - 1) / bn) > 0x7fffffffull)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "too many output tiles");
    maize::F8SkinnyParams f = {};
    f.g.c = static_cast<__nv_bfloat16 *>(c);
    f.g.ldc = ldc;
    f.g.m = m;
    f.g.n = n;
    f.g.k = k;
    f.g.tiles_m = plan.tiles_m;
    f.g.tiles_n = (n + bn - 1) / bn;
    f.g.c_vec_ok = (ldc % 8 == 0 && aligned(c, 16)) ? 1u : 0u;
    f.g.pdl = ctx->pdl;
    f.g.status = ctx->d_status;
    f.g.timeout_ns = ctx->timeout_ns;
    f.sa = sa;
    f.sb = sb;
    f.ld_sa = ld_sa;
    f.ld_sb = ld_sb;
    f.bn = bn;
    CUtensorMap ta, tb;
    maize_status_t st;
    if ((st = byte_map(ctx, &ta, a, m, k, lda, m < 128 ? m : 128)) != MAIZE_OK || (st = byte_map(ctx, &tb, b, n, k, ldb, bn)) != MAIZE_OK)
        return st;
    const int slot = maize::kAttrE4m3Skinny;
    const bool two = plan.parts == 2;
    if (plan.copies == 1)
        return two ? launch_skinny<1, 2, 6>(ctx, slot, plan.clusters, ta, tb, f, stream)
                   : launch_skinny<1, 4, 5>(ctx, slot + 1, plan.clusters, ta, tb, f, stream);
    if (plan.copies == 2)
        return two ? launch_skinny<2, 2, 4>(ctx, slot + 2, plan.clusters, ta, tb, f, stream)
                   : launch_skinny<2, 4, 3>(ctx, slot + 3, plan.clusters, ta, tb, f, stream);
    return two ? launch_skinny<4, 2, 4>(ctx, slot + 4, plan.clusters, ta, tb, f, stream)
               : launch_skinny<4, 4, 4>(ctx, slot + 5, plan.clusters, ta, tb, f, stream);
}

}  // namespace

extern "C" {

maize_status_t maize_quantize_e4m3(maize_ctx_t *ctx, const void *x, uint64_t ldx, uint32_t rows, uint32_t cols,
                                   uint32_t block_rows, void *q, uint64_t ldq, void *scales, uint64_t ld_scales,
                                   void *cuda_stream)
{
    if (!ctx)
        return MAIZE_ERR_INVALID_ARG;
    ctx->err.clear();
    if (block_rows != 1 && block_rows != maize::kQuantBlock)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "block_rows must be 1 or 128");
    if (rows == 0 || cols == 0)
        return MAIZE_OK;
    if (!x || !q || !scales)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "null pointer");
    if (!aligned(x, 2) || !aligned(scales, 4))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "x must be 2-byte and scales 4-byte aligned");
    if (rows > maize::kMaxDim || cols > maize::kMaxDim)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "rows or cols beyond the kernel's range");
    const uint64_t across = (uint64_t(cols) + 127) / 128;
    if (ldx < cols || ldq < cols || ld_scales < across)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "a leading dimension is smaller than its row");
    maize::QuantParams p = {};
    p.x = static_cast<const __nv_bfloat16 *>(x);
    p.ldx = ldx;
    p.q = static_cast<uint8_t *>(q);
    p.ldq = ldq;
    p.scales = static_cast<float *>(scales);
    p.ld_scales = ld_scales;
    p.rows = rows;
    p.cols = cols;
    p.pdl = ctx->pdl;
    // rows of X that loads of 16 bytes take as they are; rows of Q for stores of 16 bytes
    const bool xvec = ldx % 8 == 0 && aligned(x, 16), qvec = xvec && ldq % 16 == 0 && aligned(q, 16);
    DeviceGuard guard(ctx->device);
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    if (block_rows == 1) {
        // A call that does not fill the SMs gives each warp four blocks; a larger one runs of eight (sixteen where the ends of
        // a run cost more).  More CTAs than fit at a time even out the last round: 8191 x 8191 takes 56 us with 16 per SM, 70
        // with the 5 that fit; 8192 x 8192 takes 34 with either.
        const uint64_t blocks = uint64_t(rows) * across, sms = uint64_t(ctx->sm_count);
        const bool small = blocks <= sms * 6 * 32;
        const uint32_t run = small ? 4 : (qvec ? 8 : 16);
        const uint64_t want = (blocks + run * 8 - 1) / (run * 8), cap = sms * 16;
        const uint32_t grid = static_cast<uint32_t>(want < cap ? want : cap);
        auto kernel = xvec ? (qvec ? (small ? maize::quantize_rows_kernel<true, true, 1> : maize::quantize_rows_kernel<true, true, 2>)
                                   : (small ? maize::quantize_rows_kernel<true, false, 1> : maize::quantize_rows_kernel<true, false, 4>))
                           : (small ? maize::quantize_rows_kernel<false, false, 1> : maize::quantize_rows_kernel<false, false, 4>);
        return maize::launch(ctx, -1, kernel, grid, 256, 0, stream, p);
    }
    const uint64_t blocks = (uint64_t(rows) + 127) / 128 * across;
    if (blocks > 0x7fffffffull)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "too many blocks");
    auto kernel = xvec ? (qvec ? maize::quantize_blocks_kernel<true, true> : maize::quantize_blocks_kernel<true, false>)
                       : maize::quantize_blocks_kernel<false, false>;
    return maize::launch(ctx, -1, kernel, static_cast<uint32_t>(blocks), 256, 0, stream, p);
}

maize_status_t maize_gemm_e4m3(maize_ctx_t *ctx, const void *a, uint64_t lda, const void *a_scales, uint64_t ld_a_scales,
                               const void *b, uint64_t ldb, const void *b_scales, uint64_t ld_b_scales, void *c,
                               uint64_t ldc, uint32_t m, uint32_t n, uint32_t k, void *cuda_stream)
{
    if (!ctx)
        return MAIZE_ERR_INVALID_ARG;
    ctx->err.clear();
    if (m == 0 || n == 0)
        return MAIZE_OK;
    if (!c)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "C pointer is null");
    if (ldc < n)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "ldc is smaller than N");
    if (!aligned(c, 2))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "C must be 2-byte aligned");
    if (m > maize::kMaxDim || n > maize::kMaxDim || k > maize::kMaxDim)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "a dimension is beyond the kernel's range");
    DeviceGuard guard(ctx->device);
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    if (k == 0) {
        const cudaError_t e = cudaMemset2DAsync(c, ldc * 2, 0, size_t(n) * 2, m, stream);
        return e == cudaSuccess ? MAIZE_OK : fail_cuda(ctx, "cudaMemset2DAsync", e);
    }
    if (!a || !b || !a_scales || !b_scales)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "an operand or scale pointer is null");
    const uint64_t kblocks = (uint64_t(k) + 127) / 128;
    if (lda < k || ldb < k || ld_a_scales < kblocks || ld_b_scales < kblocks)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "a leading dimension is smaller than its row");
    if (!aligned(a_scales, 4) || !aligned(b_scales, 4))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "scales must be 4-byte aligned");
    if (k % 16 != 0 || lda % 16 != 0 || ldb % 16 != 0)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "K, lda and ldb must be multiples of 16 (16-byte TMA row pitch)");
    if (!aligned(a, 16) || !aligned(b, 16))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "A and B must be 16-byte aligned");
    if (lda >= (1ull << 40) || ldb >= (1ull << 40))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "row pitch beyond the TMA limit of 2^40 bytes");
    // Few rows of A, or few tiles: K over a cluster.  The other kernel takes 0.55 us for a k-block of a 256 x 256 tile and about
    // 1.5 us more for a tile's end.  128 x 8192 x 2048: 10.7 us over clusters, 12.4 in pairs; 128 x 16384 x 4096: 27.8, 20.9.
    const uint32_t ctas = maize::persistent_grid(ctx, 0xffffffffull, 1), kb = static_cast<uint32_t>(kblocks);
    SkinnyPlan plan = skinny_plan(ctx, 2, m, n, kb);
    const SkinnyPlan four = skinny_plan(ctx, 4, m, n, kb);
    if (ctx->k_parts == 0 ? four.cost < plan.cost : ctx->k_parts >= 4)
        plan = four;
    const uint64_t pair_tiles = ((uint64_t(m) + 255) / 256) * ((uint64_t(n) + 255) / 256), pairs = ctas / 2 ? ctas / 2 : 1;
    const double pair_cost = double((pair_tiles + pairs - 1) / pairs) * (kb * 0.55 + 1.5);
    if (ctx->k_parts == 0 ? plan.cost < pair_cost : ctx->k_parts != 1)
        return skinny(ctx, plan, a, lda, static_cast<const float *>(a_scales), ld_a_scales, b, ldb, static_cast<const float *>(b_scales),
                      ld_b_scales, c, ldc, m, n, k, stream);
    CUtensorMap ta, tb, tc;
    maize_status_t st;
    if ((st = byte_map(ctx, &ta, a, m, k, lda, maize::kBlockM)) != MAIZE_OK ||
        (st = byte_map(ctx, &tb, b, n, k, ldb, 128)) != MAIZE_OK)
        return st;
    memset(&tc, 0, sizeof tc);
    maize::F8Params f = {};
    maize::GemmParams &p = f.g;
    p.c = static_cast<__nv_bfloat16 *>(c);
    p.ldc = ldc;
    p.m = m;
    p.n = n;
    p.k = k;
    p.tiles_m = static_cast<uint32_t>((uint64_t(m) + 255) / 256);
    p.tiles_n = static_cast<uint32_t>((uint64_t(n) + 255) / 256);
    p.group_m = (ctx->group_rows != 0 ? ctx->group_rows : 2048u) / 256u;
    if (p.group_m == 0)
        p.group_m = 1;
    p.serpentine = ctx->serpentine;
    p.pdl = ctx->pdl;
    p.status = ctx->d_status;
    p.timeout_ns = ctx->timeout_ns;
    f.sa = static_cast<const float *>(a_scales);
    f.sb = static_cast<const float *>(b_scales);
    f.ld_sa = ld_a_scales;
    f.ld_sb = ld_b_scales;
    const bool c_rows_aligned = ldc % 8 == 0 && aligned(c, 16);
    p.c_vec_ok = c_rows_aligned ? 1u : 0u;
    if (ctx->tma_store && c_rows_aligned && n % 8 == 0 && ldc * 2 < (1ull << 40)) {
        p.c_tma_ok = maize::matrix_map(ctx, &tc, c, m, n, ldc, 32) == MAIZE_OK;
        ctx->err.clear();
    }
    const uint64_t tiles = uint64_t(p.tiles_m) * p.tiles_n;
    if (tiles > 0x7fffffffull)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "too many output tiles");
    const uint32_t grid = maize::persistent_grid(ctx, tiles, 2);
    return maize::launch(ctx, maize::kAttrE4m3, maize::gemm_e4m3_sm100_2cta<5>, grid, maize::kF8Threads,
                         maize::F8SmemLayout<5>::kDynamicBytes, stream, ta, tb, tc, f);
}

}  // extern "C"
