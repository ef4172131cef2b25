// The context behind maize_ctx_t and what every host file of the library needs with it: the device guard, the error
// text, the tensor-map encoder's type.
#pragma once
#include "../../include/maize_gemm.h"

#include <cuda_runtime.h>

#include <string>

#include "gemm_common.cuh"

namespace maize {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

constexpr int kMaxVariants = 16;        // room for the kernel variants' "attribute set" flags
constexpr uint32_t kMaxChainLanes = 4;  // streams maize_chain_forward may spread its chunks over
constexpr int kMaxHostSlabs = 16;       // row slabs of A / C that the host entry point pipelines over PCIe

class DeviceGuard {
public:
    explicit DeviceGuard(int device) : prev_(-1), changed_(false)
    {
        if (cudaGetDevice(&prev_) == cudaSuccess && prev_ != device) {
            changed_ = cudaSetDevice(device) == cudaSuccess;
        }
    }
    ~DeviceGuard()
    {
        if (changed_)
            cudaSetDevice(prev_);
    }

private:
    int prev_;
    bool changed_;
};

}  // namespace maize

struct maize_ctx {
    int device = 0;
    int sm_count = 0;
    maize::DeviceStatus *d_status = nullptr;
    maize::DeviceStatus *h_status = nullptr;  // pinned
    uint64_t timeout_ns = 2000000000ull;
    int force_kernel = 0;
    int last_kernel = 0;             // public id of the GEMM kernel the last call launched
    int max_ctas = 0;
    uint32_t debug_flags = 0;
    uint32_t group_rows = 0;         // rows of A scheduled together; 0 = by kernel (see tile_group_rows)
    uint32_t pdl = 1;       // launch the GEMM kernels with programmatic stream serialization
    uint32_t b_static = 0;  // the caller guarantees that nothing earlier in the stream writes B (weights)
    uint32_t push_threads = 512;  // threads per CTA of the copy kernels of the multi-GPU path
    uint32_t c_evict_first = 1;   // TMA stores of C carry an evict-first L2 hint
    uint64_t wide_max_gflop = 1000000;  // largest GEMM (2MNK / 1e9) that takes the wide tile
    uint32_t wide_tile = 1;       // use the 256 x 512 pair tile where it suits (long K, full rounds, about a millisecond of work)
    uint32_t tma_store = 1;       // tiled kernels: C through shared memory and TMA stores when its rows are 16-byte aligned
    uint32_t serpentine = 1;      // odd groups of row-blocks sweep the column-blocks backwards
    uint32_t tma_promotion = 3;   // CUtensorMapL2promotion of the operand maps: 0 none, 1 64 B, 2 128 B, 3 256 B
    uint32_t k_parts = 0;         // CTAs that share a tile's K in the grouped and e4m3 products; 0 = by size
    uint32_t tail_split = 1;      // split the last partial round of pair tiles along K when pairs would idle
    uint32_t chain_stagger = 1;   // two lanes on a source that is all there: offset them by half a chunk
    uint32_t chain_streams = 2;   // 2: maize_chain_forward alternates chunks between the caller's stream and a helper
    cudaStream_t chain_helper[maize::kMaxChainLanes] = {};  // lanes 1 .. L-1 of maize_chain_forward (lane 0 is the caller's stream)
    cudaEvent_t chain_ev_fork = nullptr;             // the caller's stream as of the call
    cudaEvent_t chain_ev_pub[maize::kMaxChainLanes] = {};   // "chunk published" per lane
    cudaEvent_t chain_ev_part[maize::kMaxChainLanes] = {};  // pieces of the first chunk sent (offsets the lanes)
    uint64_t launches = 0;
    maize::EncodeTiledFn encode = nullptr;
    void *staging = nullptr;  // device staging for the *_host entry point
    size_t staging_bytes = 0;
    // B of the last *_host call, still in the staging area: re-used instead of re-uploaded under "b_static"
    const void *host_b_ptr = nullptr;
    uint32_t host_b_rows = 0, host_b_cols = 0;
    char *host_b_dev = nullptr;
    void *repack = nullptr;  // scratch for operands copied to a 128-byte-aligned pitch ("repack_bytes")
    size_t repack_bytes = 0;
    const void *repack_b_ptr = nullptr;  // B whose aligned-pitch copy sits at the front of `repack` ("b_static" only)
    uint32_t repack_b_rows = 0, repack_b_cols = 0;
    uint64_t repack_b_ld = 0;
    // helper streams and events of the *_host entry point (created on first use)
    cudaStream_t copy_in = nullptr, copy_out = nullptr;
    cudaEvent_t ev_start = nullptr, ev_done = nullptr;
    cudaEvent_t ev_in[maize::kMaxHostSlabs] = {}, ev_gemm[maize::kMaxHostSlabs] = {};
    bool attr_set[maize::kMaxVariants] = {};
    bool attr_set_kn[maize::kMaxVariants] = {};  // the same for the K x N (MN-major B) instantiations
    bool attr_experts[24] = {};                  // the same for the kernels of maize_experts.cu and maize_e4m3.cu
    uint32_t clusters_at_once[2] = {0, 0};  // clusters of four, of eight CTAs that the device runs at a time; 0: not asked yet
    float *d_partials = nullptr;        // stream-K scratch of the skinny kernels
    unsigned int *d_counters = nullptr;  // arrival counters, zero between launches
    unsigned int *d_push_counter = nullptr;  // [0]: CTA arrivals of the multicast push; [16 + p]: of the scatter per rank
    unsigned long long *d_profile = nullptr;  // kProfileSlots counters per CTA, allocated when "profile" is set
    int profile_ctas = 0;                      // CTAs of the last profiled launch
    std::string err;
};

namespace maize {

inline maize_status_t fail(maize_ctx_t *ctx, maize_status_t st, const std::string &msg)
{
    if (ctx)
        ctx->err = msg;
    return st;
}

inline maize_status_t fail_cuda(maize_ctx_t *ctx, const char *what, cudaError_t e)
{
    return fail(ctx, MAIZE_ERR_CUDA, std::string(what) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
}

}  // namespace maize
