// C ABI of the grouped ("expert") products (declared in include/maize_gemm.h): argument validation, tensor maps over
// stacks of matrices, launches.  The sizes of the groups are known on the device only; what the host checks is
// everything else.
#include "../../include/maize_gemm.h"

#include <cstring>

#include "maize_host.cuh"
#include "gemm_sm100_grouped.cuh"
#include "gemm_sm100_grouped_split.cuh"
#include "gemm_sm100_grouped_wgrad.cuh"
#include "gemm_sm100_grouped_wgrad_split.cuh"

namespace {

using maize::DeviceGuard;
using maize::fail;
using maize::fail_cuda;
using maize::GroupedParams;

using maize::aligned;
using maize::kMaxDim;
using maize::launch;
using maize::matrix_map;
using maize::persistent_grid;
using maize::stack_map;

// What the three grouped entry points check alike.
maize_status_t check_groups(maize_ctx_t *ctx, const void *offsets, uint32_t groups, uint32_t rows)
{
    if (!offsets || !aligned(offsets, 4))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "offsets must be a 4-byte aligned device array of groups + 1 integers");
    if (groups > maize::kGroupedMaxGroups)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "more than 1024 groups");
    if (rows > kMaxDim)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "too many rows for 32-bit offsets");
    return MAIZE_OK;
}

// A stack of row-major matrices [rows x cols]: the matrices may not overlap.
bool stack_ok(uint32_t count, uint64_t stride, uint64_t rows, uint64_t cols, uint64_t ld)
{
    return count <= 1 || rows == 0 || stride >= (rows - 1) * ld + cols;
}

uint32_t clusters_of(maize_ctx_t *ctx, uint32_t parts)
{
    if (parts == 8)
        return maize::clusters_at_once(ctx, 8, maize::gemm_bf16_sm100_grouped_split<false, 8, 7>, maize::kNumThreads,
                                       maize::GroupedSplitLayout<8, 7>::kDynamicBytes);
    return maize::clusters_at_once(ctx, parts, maize::gemm_bf16_sm100_grouped_split<false, 4, 7>, maize::kNumThreads,
                                   maize::GroupedSplitLayout<4, 7>::kDynamicBytes);
}

// What sharing a tile's sum among `parts` CTAs costs, in microseconds beyond what every call takes, for comparison only.
struct SplitCost {
    double end;    // of the last tile
    double least;  // of any other tile: behind a short sum the one before is not yet stored
};

double split_cost(const SplitCost &c, uint64_t tiles, uint64_t at_a_time, double sum)
{
    const uint64_t rounds = (tiles + at_a_time - 1) / at_a_time;
    return c.end + sum + double(rounds - 1) * (sum > c.least ? sum : c.least);
}

// CTAs that share a tile's K, or 1 for the kernel that gives a pair whole tiles.  Both are reckoned with the most tiles that
// the rows can make, 0.27 us for a k-block, and what was measured of the tiles' ends; neither is faster than the weights come.
// Eight rows for five experts, 144 x 6936: 8 us in eight parts, 35 whole; 39 rows for one, 4096 x 4096: 10.6 in four parts, 20
// in eight (two rounds), 22 whole; 32 rows for 16 experts, 4096 x 2048: 48 in two parts, 65 in four, 46 to 50 whole.
uint32_t split_parts(maize_ctx_t *ctx, uint32_t rows, uint32_t groups, uint32_t n, uint32_t k)
{
    if (ctx->k_parts != 0)
        return ctx->k_parts;
    const uint64_t with_rows = rows < groups ? rows : groups, kb = (uint64_t(k) + 63) / 64;
    const double weights = double(with_rows) * n * k * 2 / 6.2e6;
    const SplitCost costs[4] = {{1.0, 2.1}, {1.6, 2.6}, {1.4, 2.1}, {1.3, 3.6}};
    const uint64_t pair_tiles = (rows / maize::kGroupedTileRows + with_rows) * ((uint64_t(n) + 255) / 256);
    double best = split_cost(costs[0], pair_tiles, clusters_of(ctx, 2), double(kb) * 0.27);
    const uint64_t tiles = (rows / maize::kSplitTileRows + with_rows) * ((uint64_t(n) + 127) / 128);
    uint32_t parts = 1;
    for (uint32_t i = 1; i <= 3 && best > weights; ++i) {
        const uint32_t s = 1u << i;
        const double cost = split_cost(costs[i], tiles, clusters_of(ctx, s), double((kb + s - 1) / s) * 0.27);
        if (cost < best) {
            best = cost;
            parts = s;
        }
    }
    return parts;
}

template <bool W_KN, uint32_t S, uint32_t STAGES>
maize_status_t launch_split(maize_ctx_t *ctx, const maize::RowMaps &ta, const CUtensorMap &tw, const GroupedParams &p,
                            cudaStream_t stream)
{
    const uint64_t tiles = (p.rows / maize::kSplitTileRows + uint64_t(p.rows < p.groups ? p.rows : p.groups)) *
                           ((uint64_t(p.n) + maize::kSplitTileCols - 1) / maize::kSplitTileCols);
    const uint32_t most = clusters_of(ctx, S), clusters = tiles < most ? static_cast<uint32_t>(tiles) : most;
    const int slot = maize::kAttrGroupedSplit + (W_KN ? 3 : 0) + (S == 2 ? 0 : (S == 4 ? 1 : 2));
    return maize::launch_clusters(ctx, slot, maize::gemm_bf16_sm100_grouped_split<W_KN, S, STAGES>, clusters * S, S,
                                  maize::kNumThreads, maize::GroupedSplitLayout<S, STAGES>::kDynamicBytes, stream, ta, tw, p);
}

// The same choice for the weight gradient, whose sum runs over a group's rows: reckoned with the mean group, half as long again
// where every tile has a pair or cluster to itself and the longest group decides.  11186 rows of one group, 136 x 544: 15 us in
// eight parts, 21 in four, 61 whole; 16384 rows, 4096 x 4096: 417 whole, 751 in two; 290 rows, 112 x 32: 6 whole, 10.9 in two.
uint32_t wgrad_parts(maize_ctx_t *ctx, uint32_t rows, uint32_t groups, uint32_t n, uint32_t k)
{
    if (ctx->k_parts != 0)
        return ctx->k_parts;
    const uint64_t mean = (uint64_t(rows) / groups + 63) / 64;
    auto blocks = [](uint64_t size, uint64_t tile) { return (size + tile - 1) / tile; };
    auto sum = [&](uint64_t tiles, uint64_t at_a_time, uint64_t parts) {
        return double(blocks(groups > 1 && tiles <= at_a_time ? mean + mean / 2 : mean, parts)) * 0.35;
    };
    const SplitCost costs[4] = {{1.0, 2.7}, {5.0, 4.5}, {4.5, 3.5}, {3.9, 4.0}};
    const uint64_t pair_tiles = groups * blocks(n, 256) * blocks(k, 256), pairs = clusters_of(ctx, 2);
    double best = split_cost(costs[0], pair_tiles, pairs, sum(pair_tiles, pairs, 1));
    const uint64_t tiles = groups * blocks(n, maize::kWgradSplitTile) * blocks(k, maize::kWgradSplitTile);
    uint32_t parts = 1;
    for (uint32_t i = 1; i <= 3; ++i) {
        const uint32_t s = 1u << i, at_a_time = clusters_of(ctx, s);
        const double cost = split_cost(costs[i], tiles, at_a_time, sum(tiles, at_a_time, s));
        if (cost < best) {
            best = cost;
            parts = s;
        }
    }
    return parts;
}

template <uint32_t S, uint32_t STAGES>
maize_status_t launch_wgrad_split(maize_ctx_t *ctx, const CUtensorMap &tdc, const CUtensorMap &ta, const GroupedParams &p,
                                  cudaStream_t stream)
{
    const uint64_t tiles = uint64_t(p.groups) * ((uint64_t(p.n) + 127) / 128) * ((uint64_t(p.k) + 127) / 128);
    if (tiles > 0x7fffffffull)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "too many output tiles");
    const uint32_t most = clusters_of(ctx, S), clusters = tiles < most ? static_cast<uint32_t>(tiles) : most;
    const int slot = maize::kAttrWgradSplit + (S == 2 ? 0 : (S == 4 ? 1 : 2));
    return maize::launch_clusters(ctx, slot, maize::gemm_bf16_sm100_grouped_wgrad_split<S, STAGES>, clusters * S, S,
                                  maize::kWgradSplitThreads, maize::WgradSplitLayout<S, STAGES>::kDynamicBytes, stream, tdc, ta, p);
}

maize_status_t grouped_impl(maize_ctx_t *ctx, const void *a, uint64_t lda, const void *b, uint64_t ldb, uint64_t b_stride,
                            void *c, uint64_t ldc, const void *offsets, uint32_t groups, uint32_t rows, uint32_t n,
                            uint32_t k, cudaStream_t stream, bool b_kn)
{
    if (!ctx)
        return MAIZE_ERR_INVALID_ARG;
    ctx->err.clear();
    if (rows == 0 || n == 0 || groups == 0)
        return MAIZE_OK;
    maize_status_t st = check_groups(ctx, offsets, groups, rows);
    if (st != MAIZE_OK)
        return st;
    if (!c)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "C pointer is null");
    if (ldc < n)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "ldc is smaller than N");
    if (!aligned(c, 2))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "C must be 2-byte aligned");
    if (n > kMaxDim || k > kMaxDim)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "N or K beyond the kernel's range");
    GroupedParams p = {};
    p.c = static_cast<__nv_bfloat16 *>(c);
    p.ldc = ldc;
    p.offsets = static_cast<const int32_t *>(offsets);
    p.groups = groups;
    p.rows = rows;
    p.n = n;
    p.k = k;
    p.c_pair_ok = (ldc % 2 == 0 && aligned(c, 4)) ? 1u : 0u;
    p.pdl = ctx->pdl;
    p.status = ctx->d_status;
    p.timeout_ns = ctx->timeout_ns;
    DeviceGuard guard(ctx->device);
    if (k == 0) {
        maize::grouped_zero_rows_kernel<<<static_cast<uint32_t>(ctx->sm_count), 256, 0, stream>>>(p);
        ctx->launches += 1;
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? MAIZE_OK : fail_cuda(ctx, "kernel launch", e);
    }
    if (!a || !b)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "A or B pointer is null");
    if (lda < k || ldb < (b_kn ? n : k))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "lda/ldb is smaller than the row length");
    if (!stack_ok(groups, b_stride, b_kn ? k : n, b_kn ? n : k, ldb))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "the matrices of B overlap: b_stride is smaller than a matrix");
    if (groups == 1)
        b_stride = uint64_t(b_kn ? k : n) * ldb;  // not used for addressing; the map wants a valid pitch
    if (lda % 8 != 0 || ldb % 8 != 0 || b_stride % 8 != 0 || (!b_kn && k % 8 != 0))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "K, lda, ldb and b_stride must be multiples of 8 (16-byte TMA pitch)");
    if (!aligned(a, 16) || !aligned(b, 16))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "A and B must be 16-byte aligned");
    if (lda * 2 >= (1ull << 40) || ldb * 2 >= (1ull << 40) || b_stride * 2 >= (1ull << 40))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "pitch beyond the TMA limit of 2^40 bytes");

    const uint32_t parts = split_parts(ctx, rows, groups, n, k);
    // the boxes that tiles of these rows can need: a CTA of a pair brings in half a tile's rows, one of a split tile all
    const uint32_t longest = parts > 1 ? rows : (rows + 31) / 32 * 16;
    maize::RowMaps ta = {};
    for (uint32_t i = 0; i < (parts > 1 ? 3u : 4u) && (i == 0 || (8u << i) < longest); ++i)
        if ((st = matrix_map(ctx, &ta.box[i], a, rows, k, lda, 16u << i)) != MAIZE_OK)
            return st;
    CUtensorMap tw;
    const CUtensorMapL2promotion promotion = static_cast<CUtensorMapL2promotion>(ctx->tma_promotion);
    st = b_kn ? stack_map(ctx, &tw, b, groups, k, n, ldb, b_stride, maize::kBlockK, promotion)
              : stack_map(ctx, &tw, b, groups, n, k, ldb, b_stride, maize::kBlockM, promotion);
    if (st != MAIZE_OK)
        return st;
    if (parts == 8)
        return b_kn ? launch_split<true, 8, 7>(ctx, ta, tw, p, stream) : launch_split<false, 8, 7>(ctx, ta, tw, p, stream);
    if (parts == 4)
        return b_kn ? launch_split<true, 4, 7>(ctx, ta, tw, p, stream) : launch_split<false, 4, 7>(ctx, ta, tw, p, stream);
    if (parts == 2)
        return b_kn ? launch_split<true, 2, 7>(ctx, ta, tw, p, stream) : launch_split<false, 2, 7>(ctx, ta, tw, p, stream);

    // rows of C that TMA can store (N has to end on a 16-byte piece, see the weight gradient)
    CUtensorMap tc;
    memset(&tc, 0, sizeof tc);
    if (ctx->tma_store && n % 8 == 0 && ldc % 8 == 0 && aligned(c, 16) && ldc * 2 < (1ull << 40)) {
        p.c_tma_ok = matrix_map(ctx, &tc, c, rows, n, ldc, 32) == MAIZE_OK;
        ctx->err.clear();
    }

    const uint64_t n_blocks = (uint64_t(n) + maize::kGroupedTileCols - 1) / maize::kGroupedTileCols;
    // at most: whole row tiles plus one more in every group that has rows
    const uint64_t row_tiles = rows / maize::kGroupedTileRows + (rows < groups ? rows : groups);
    const uint32_t grid = persistent_grid(ctx, row_tiles * n_blocks, 2);
    using L = maize::GroupedSmemLayout<6>;
    return b_kn ? launch(ctx, maize::kAttrGroupedKn, maize::gemm_bf16_sm100_grouped<true, 6>, grid, maize::kGroupedThreads,
                         L::kDynamicBytes, stream, ta, tw, tc, p)
                : launch(ctx, maize::kAttrGrouped, maize::gemm_bf16_sm100_grouped<false, 6>, grid, maize::kGroupedThreads,
                         L::kDynamicBytes, stream, ta, tw, tc, p);
}

}  // namespace

extern "C" {

maize_status_t maize_grouped_gemm_bf16(maize_ctx_t *ctx, const void *a, uint64_t lda, const void *b, uint64_t ldb,
                                       uint64_t b_stride, void *c, uint64_t ldc, const void *offsets, uint32_t groups,
                                       uint32_t rows, uint32_t n, uint32_t k, void *cuda_stream)
{
    return grouped_impl(ctx, a, lda, b, ldb, b_stride, c, ldc, offsets, groups, rows, n, k,
                        static_cast<cudaStream_t>(cuda_stream), false);
}

maize_status_t maize_grouped_gemm_bf16_kn(maize_ctx_t *ctx, const void *a, uint64_t lda, const void *b, uint64_t ldb,
                                          uint64_t b_stride, void *c, uint64_t ldc, const void *offsets, uint32_t groups,
                                          uint32_t rows, uint32_t n, uint32_t k, void *cuda_stream)
{
    return grouped_impl(ctx, a, lda, b, ldb, b_stride, c, ldc, offsets, groups, rows, n, k,
                        static_cast<cudaStream_t>(cuda_stream), true);
}

maize_status_t maize_grouped_gemm_bf16_wgrad(maize_ctx_t *ctx, const void *a, uint64_t lda, const void *dc, uint64_t lddc,
                                             void *db, uint64_t lddb, uint64_t db_stride, const void *offsets,
                                             uint32_t groups, uint32_t rows, uint32_t n, uint32_t k, void *cuda_stream)
{
    if (!ctx)
        return MAIZE_ERR_INVALID_ARG;
    ctx->err.clear();
    if (n == 0 || k == 0 || groups == 0)
        return MAIZE_OK;
    maize_status_t st = check_groups(ctx, offsets, groups, rows);
    if (st != MAIZE_OK)
        return st;
    if (!db)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "DB pointer is null");
    if (lddb < k)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "lddb is smaller than K");
    if (!aligned(db, 2))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "DB must be 2-byte aligned");
    if (!stack_ok(groups, db_stride, n, k, lddb))
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "the matrices of DB overlap: db_stride is smaller than a matrix");
    if (n > kMaxDim || k > kMaxDim)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "N or K beyond the kernel's range");
    const uint64_t tiles = uint64_t(groups) * ((uint64_t(n) + 255) / 256) * ((uint64_t(k) + 255) / 256);
    if (tiles > 0x7fffffffull)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "too many output tiles");
    DeviceGuard guard(ctx->device);
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    if (rows == 0) {
        // no rows at all: every gradient is zero
        for (uint32_t g = 0; g < groups; ++g) {
            const cudaError_t e = cudaMemset2DAsync(static_cast<char *>(db) + uint64_t(g) * db_stride * 2, lddb * 2, 0,
                                                    size_t(k) * 2, n, stream);
            if (e != cudaSuccess)
                return fail_cuda(ctx, "cudaMemset2DAsync", e);
        }
        return MAIZE_OK;
    }
    if (!a || !dc)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "A or DC pointer is null");
    if (lda < k || lddc < n)
        return fail(ctx, MAIZE_ERR_INVALID_ARG, "lda/lddc is smaller than the row length");
    if (lda % 8 != 0 || lddc % 8 != 0)
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "lda and lddc must be multiples of 8 (16-byte TMA pitch)");
    if (!aligned(a, 16) || !aligned(dc, 16))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "A and DC must be 16-byte aligned");
    if (lda * 2 >= (1ull << 40) || lddc * 2 >= (1ull << 40))
        return fail(ctx, MAIZE_ERR_UNSUPPORTED, "pitch beyond the TMA limit of 2^40 bytes");
    CUtensorMap tdc, ta, tdw;
    if ((st = matrix_map(ctx, &tdc, dc, rows, n, lddc, maize::kBlockK)) != MAIZE_OK ||
        (st = matrix_map(ctx, &ta, a, rows, k, lda, maize::kBlockK)) != MAIZE_OK)
        return st;
    memset(&tdw, 0, sizeof tdw);
    if (groups == 1)
        db_stride = uint64_t(n) * lddb;
    GroupedParams p = {};
    p.c = static_cast<__nv_bfloat16 *>(db);
    p.ldc = lddb;
    p.c_stride = db_stride;
    p.offsets = static_cast<const int32_t *>(offsets);
    p.groups = groups;
    p.rows = rows;
    p.n = n;
    p.k = k;
    p.c_evict_first = ctx->c_evict_first;
    p.pdl = ctx->pdl;
    p.status = ctx->d_status;
    p.timeout_ns = ctx->timeout_ns;
    p.c_vec_ok = (lddb % 8 == 0 && db_stride % 8 == 0 && aligned(db, 16)) ? 1u : 0u;
    switch (wgrad_parts(ctx, rows, groups, n, k)) {
    case 2: return launch_wgrad_split<2, 4>(ctx, tdc, ta, p, stream);
    case 4: return launch_wgrad_split<4, 4>(ctx, tdc, ta, p, stream);
    case 8: return launch_wgrad_split<8, 4>(ctx, tdc, ta, p, stream);
    default: break;
    }
    // Rows of DB that TMA can store: a store writes whole 16-byte pieces, so K has to end on one (a K of 57 had zeros
    // written into the seven columns behind it).  A stack the driver refuses goes by plain stores too.
    if (ctx->tma_store && k % 8 == 0 && lddb % 8 == 0 && db_stride % 8 == 0 && aligned(db, 16) && lddb * 2 < (1ull << 40) &&
        db_stride * 2 < (1ull << 40)) {
        p.c_tma_ok = stack_map(ctx, &tdw, db, groups, n, k, lddb, db_stride, 32, CU_TENSOR_MAP_L2_PROMOTION_NONE) == MAIZE_OK;
        ctx->err.clear();
    }
    const uint32_t grid = persistent_grid(ctx, tiles, 2);
    return launch(ctx, maize::kAttrWgrad, maize::gemm_bf16_sm100_grouped_wgrad<5>, grid, maize::kWgradThreads,
                  maize::WgradSmemLayout<5>::kDynamicBytes, stream, tdc, ta, tdw, p);
}

}  // extern "C"
