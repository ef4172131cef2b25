// Host-side pieces of the entry points beside the dense bf16 GEMM: tensor maps over matrices and stacks of matrices, launches.
#pragma once
#include <cstdio>

#include "maize_ctx.cuh"

namespace maize {

constexpr uint32_t kMaxDim = 0x7fffff00u;  // sizes are TMA coordinates (int32); room for a tile past the end

// ctx->attr_experts slots: kernels whose shared-memory limit has been raised on the context's device
enum { kAttrGrouped = 0, kAttrGroupedKn = 1, kAttrWgrad = 2, kAttrE4m3 = 3, kAttrE4m3Skinny = 4 /* .. 9 */, kAttrGroupedSplit = 10 /* .. 15 */,
       kAttrWgradSplit = 16 /* .. 18 */ };

inline bool aligned(const void *p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

inline maize_status_t encode_map(maize_ctx_t *ctx, CUtensorMap *map, CUtensorMapDataType type, uint32_t element_bytes,
                          const void *base, uint32_t rank, const uint64_t *dims, const uint64_t *strides,
                          const uint32_t *box_dims, CUtensorMapL2promotion promotion)
{
    cuuint64_t gdim[3], gstride[2];
    cuuint32_t box[3], estride[3] = {1, 1, 1};
    for (uint32_t i = 0; i < rank; ++i) {
        gdim[i] = dims[i];
        box[i] = box_dims[i];
        if (i + 1 < rank)
            gstride[i] = strides[i] * element_bytes;
    }
    const CUresult r = ctx->encode(map, type, rank, const_cast<void *>(base), gdim, gstride, box, estride,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promotion,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS)
        return MAIZE_OK;
    char buf[160];
    snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed (CUresult %d) for %llu x %llu, ld %llu", (int)r,
             (unsigned long long)dims[1], (unsigned long long)dims[0], (unsigned long long)strides[0]);
    return fail(ctx, MAIZE_ERR_CUDA, buf);
}

// [rows x cols] bf16, boxes of box_rows x 64.
inline maize_status_t matrix_map(maize_ctx_t *ctx, CUtensorMap *map, const void *base, uint64_t rows, uint64_t cols, uint64_t ld,
                          uint32_t box_rows)
{
    const uint64_t dims[2] = {cols, rows}, strides[1] = {ld};
    const uint32_t box[2] = {kBlockK, box_rows};
    return encode_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, 2, dims, strides, box,
                      static_cast<CUtensorMapL2promotion>(ctx->tma_promotion));
}

// A stack of `count` bf16 matrices [rows x cols], `stride` elements apart, boxes of 1 x box_rows x 64.
inline maize_status_t stack_map(maize_ctx_t *ctx, CUtensorMap *map, const void *base, uint64_t count, uint64_t rows, uint64_t cols,
                         uint64_t ld, uint64_t stride, uint32_t box_rows, CUtensorMapL2promotion promotion)
{
    const uint64_t dims[3] = {cols, rows, count}, strides[2] = {ld, stride};
    const uint32_t box[3] = {kBlockK, box_rows, 1};
    return encode_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, 3, dims, strides, box, promotion);
}

// Kernels launched in clusters of `cluster` CTAs (0: as the kernel itself says).  `attr_slot` < 0: a kernel that needs no
// more shared memory than any may have.
template <typename Kernel, typename... Args>
maize_status_t launch_clusters(maize_ctx_t *ctx, int attr_slot, Kernel kernel, uint32_t grid, uint32_t cluster, uint32_t threads,
                               uint32_t smem, cudaStream_t stream, const Args &...args)
{
    if (attr_slot >= 0 && !ctx->attr_experts[attr_slot]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess)
            return fail_cuda(ctx, "cudaFuncSetAttribute(max dynamic smem)", e);
        ctx->attr_experts[attr_slot] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    if (ctx->pdl) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster != 0) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess)
        return fail_cuda(ctx, "kernel launch", e);
    ctx->launches += 1;
    return MAIZE_OK;
}

template <typename Kernel, typename... Args>
maize_status_t launch(maize_ctx_t *ctx, int attr_slot, Kernel kernel, uint32_t grid, uint32_t threads, uint32_t smem,
                      cudaStream_t stream, const Args &...args)
{
    return launch_clusters(ctx, attr_slot, kernel, grid, 0, threads, smem, stream, args...);
}

// CTAs that may run at a time, a multiple of `unit` (the cluster size), at most what `tiles` clusters need.
inline uint32_t persistent_grid(const maize_ctx_t *ctx, uint64_t tiles, uint32_t unit)
{
    uint32_t cap = static_cast<uint32_t>(ctx->sm_count);
    if (ctx->max_ctas > 0 && static_cast<uint32_t>(ctx->max_ctas) < cap)
        cap = static_cast<uint32_t>(ctx->max_ctas);
    cap /= unit;
    if (cap == 0)
        cap = 1;
    return (tiles < cap ? static_cast<uint32_t>(tiles) : cap) * unit;
}

// Clusters of `parts` = 2, 4 or 8 CTAs that may run at a time, for kernels whose CTAs have an SM to themselves.  Those of four
// and eight fit only within a GPC, and how many SMs its GPCs have differs from one part to the next: the driver is asked, once for
// a context, with one of these kernels (33 of four and 15 of eight on one B200; a sixteenth of eight waited for a whole
// wave: 6.8 -> 11.8 us).
template <typename Kernel>
uint32_t clusters_at_once(maize_ctx_t *ctx, uint32_t parts, Kernel kernel, uint32_t threads, uint32_t smem)
{
    const uint32_t ctas = persistent_grid(ctx, 0xffffffffull, 1), whole = ctas / parts ? ctas / parts : 1;
    if (parts == 2)
        return whole;
    uint32_t &known = ctx->clusters_at_once[parts == 4 ? 0 : 1];
    if (known == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<uint32_t>(ctx->sm_count) / parts * parts);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = parts;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();  // an estimate will do: the answer is for speed only
            n = ctx->sm_count / static_cast<int>(parts) * 7 / 8;
        }
        known = n < 1 ? 1u : static_cast<uint32_t>(n);
    }
    return known < whole ? known : whole;
}

}  // namespace maize
