// bf16 -> e4m3 with one power-of-two scale for each block of 1 x 128 or 128 x 128 elements.
//
//     s = 2^p, p = the smallest integer >= -126 with max|x| <= 448 * 2^p  (max over the block's finite elements; 1 if all 0)
//     q = e4m3(x / s), round to nearest even; what is not finite becomes NaN
//
// A power of two makes x / s exact, so the conversion to e4m3 is the only rounding, and it costs no precision: e4m3 keeps
// three mantissa bits at any magnitude down to 2^-6, 14 binades below the largest.
//
// Bound: HBM; 2 bytes read and 1 written per element.  A block's elements stay in registers between the maximum and the
// conversion, so the input is read once.
#pragma once
#include "gemm_common.cuh"

namespace maize {

constexpr uint32_t kQuantBlock = 128;

struct QuantParams {
    const __nv_bfloat16 *x;
    uint64_t ldx;
    uint8_t *q;
    uint64_t ldq;
    float *scales;
    uint64_t ld_scales;
    uint32_t rows, cols;
    uint32_t pdl;
};

// max|x| (fp32, finite) -> the scale's and its inverse's bits.  448 = 1.75 * 2^8: p = exponent - 8, one more where the
// mantissa is above 1.75.
__device__ __forceinline__ void block_scale(float amax, float &scale, float &inverse)
{
    const uint32_t bits = __float_as_uint(amax);
    int32_t e = static_cast<int32_t>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < 1 ? 1 : e;
    e = amax > 0.0f ? e : 127;
    scale = __uint_as_float(static_cast<uint32_t>(e) << 23);
    inverse = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Eight bf16 in four words.
struct Eight {
    uint32_t w[4];
};

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Largest finite magnitude; `seen_inf` where an element is infinite or NaN (the caller then clears those).
__device__ __forceinline__ float eight_amax(const Eight &v, bool &odd)
{
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = fabsf(bf16_lo(v.w[i])), b = fabsf(bf16_hi(v.w[i]));
        const bool fa = a <= 3.4e38f, fb = b <= 3.4e38f;  // false for infinities and NaN: bf16's largest is 3.39e38
        odd |= !(fa && fb);
        m = fmaxf(m, fa ? a : 0.0f);
        m = fmaxf(m, fb ? b : 0.0f);
    }
    return m;
}

__device__ __forceinline__ float scaled(float x, float inverse, bool odd)
{
    const float v = x * inverse;
    return odd && !(fabsf(x) <= 3.4e38f) ? __uint_as_float(0x7fffffffu) : v;
}

__device__ __forceinline__ uint2 eight_convert(const Eight &v, float inverse, bool odd)
{
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = to_e4m3x2(scaled(bf16_lo(v.w[i]), inverse, odd), scaled(bf16_hi(v.w[i]), inverse, odd));
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// Elements col .. col+7 of a row, zeros past the end.
template <bool VEC>
__device__ __forceinline__ Eight load_eight(const __nv_bfloat16 *row, uint32_t col, uint32_t cols)
{
    Eight v;
    if (VEC && col + 8 <= cols) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(row + col));
        v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
        return v;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t c = col + 2 * i;
        const uint32_t lo = c < cols ? __ldg(reinterpret_cast<const uint16_t *>(row + c)) : 0u;
        const uint32_t hi = c + 1 < cols ? __ldg(reinterpret_cast<const uint16_t *>(row + c + 1)) : 0u;
        v.w[i] = lo | (hi << 16);
    }
    return v;
}

template <bool VEC>
__device__ __forceinline__ void store_eight(uint8_t *row, uint32_t col, uint32_t cols, uint2 b)
{
    if (VEC && col + 8 <= cols) {
        *reinterpret_cast<uint2 *>(row + col) = b;
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (col + i < cols)
            row[col + i] = static_cast<uint8_t>((i < 4 ? b.x : b.y) >> (8 * (i & 3u)));
}

// 1 x 128 blocks: 16 lanes of a warp hold one block, eight elements each.
template <bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p)
{
    if (p.pdl) {
        ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t across = (p.cols + kQuantBlock - 1) / kQuantBlock;
    const uint64_t blocks = static_cast<uint64_t>(p.rows) * across;
    const uint32_t lane16 = threadIdx.x & 15u;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * (blockDim.x / 16);
    const uint64_t first = (static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 16;
    // whole warps go round: the shuffles below need both halves of one
    const uint64_t rounds = (blocks + step - 1) / step;
    for (uint64_t i = 0; i < rounds; ++i) {
        const uint64_t b = first + i * step;
        const bool mine = b < blocks;
        const uint32_t row = mine ? static_cast<uint32_t>(b / across) : 0u;
        const uint32_t blk = mine ? static_cast<uint32_t>(b - static_cast<uint64_t>(row) * across) : 0u;
        const uint32_t col = blk * kQuantBlock + lane16 * 8u;
        Eight v{};
        if (mine)
            v = load_eight<VEC>(p.x + static_cast<uint64_t>(row) * p.ldx, col, p.cols);
        bool odd = false;
        float m = eight_amax(v, odd);
#pragma unroll
        for (uint32_t d = 8; d > 0; d >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        float scale, inverse;
        block_scale(m, scale, inverse);
        if (mine) {
            store_eight<VEC>(p.q + static_cast<uint64_t>(row) * p.ldq, col, p.cols, eight_convert(v, inverse, odd));
            if (lane16 == 0)
                p.scales[static_cast<uint64_t>(row) * p.ld_scales + blk] = scale;
        }
    }
}

// 128 x 128 blocks: one CTA per block, 16 threads per row, eight rows per thread.
template <bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantParams p)
{
    __shared__ float warp_max[8];
    if (p.pdl) {
        ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t across = (p.cols + kQuantBlock - 1) / kQuantBlock;
    const uint32_t down = blockIdx.x / across, blk = blockIdx.x - down * across;
    const uint32_t col = blk * kQuantBlock + (threadIdx.x & 15u) * 8u;
    const uint32_t row0 = down * kQuantBlock + threadIdx.x / 16u;
    Eight v[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = row0 + 16u * i;
        v[i] = Eight{};
        if (row < p.rows)
            v[i] = load_eight<VEC>(p.x + static_cast<uint64_t>(row) * p.ldx, col, p.cols);
    }
    bool odd = false;
    float m = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        m = fmaxf(m, eight_amax(v[i], odd));
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31u) == 0)
        warp_max[threadIdx.x / 32u] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        m = fmaxf(m, warp_max[i]);
    float scale, inverse;
    block_scale(m, scale, inverse);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = row0 + 16u * i;
        if (row < p.rows)
            store_eight<VEC>(p.q + static_cast<uint64_t>(row) * p.ldq, col, p.cols, eight_convert(v[i], inverse, odd));
    }
    if (threadIdx.x == 0)
        p.scales[static_cast<uint64_t>(down) * p.ld_scales + blk] = scale;
}

}  // namespace maize
