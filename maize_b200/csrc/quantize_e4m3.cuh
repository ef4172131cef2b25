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

// Largest magnitude of a block as bf16 bits (finite) -> the scale and its inverse.  448 = 1.75 * 2^8: the scale's exponent
// is the magnitude's less 8, one more where the mantissa is above 1.75.
__device__ __forceinline__ void block_scale(uint32_t top, float &scale, float &inverse)
{
    int32_t e = static_cast<int32_t>(top >> 7) - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0);
    e = e < 1 ? 1 : e;
    e = top != 0u ? e : 127;
    scale = __uint_as_float(static_cast<uint32_t>(e) << 23);
    inverse = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t max_s16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.s16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Eight bf16 in four words.
struct Eight {
    uint32_t w[4];
};

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

constexpr uint32_t kBf16Inf = 0x7f80u;

// The eight one by one, where one of them is infinite or NaN: the largest finite magnitude, and the conversion with NaN in
// their places (the conversion instruction would saturate infinities).  Out of line: nearly no data comes here.
static __device__ __noinline__ uint32_t odd_eight_top(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3)
{
    const uint32_t w[4] = {w0, w1, w2, w3};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
        m = max(m, max(lo < kBf16Inf ? lo : 0u, hi < kBf16Inf ? hi : 0u));
    }
    return m;
}

static __device__ __noinline__ uint2 odd_eight_convert(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, float inverse)
{
    const uint32_t w[4] = {w0, w1, w2, w3};
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float nan = __uint_as_float(0x7fffffffu);
        h[i] = to_e4m3x2((w[i] & 0x7fffu) >= kBf16Inf ? nan : bf16_lo(w[i]) * inverse,
                         ((w[i] >> 16) & 0x7fffu) >= kBf16Inf ? nan : bf16_hi(w[i]) * inverse);
    }
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// Largest finite magnitude of the eight, as bf16 bits (they order like integers); `odd` is set where one is not finite.
__device__ __forceinline__ uint32_t eight_top(const Eight &v, bool &odd)
{
    constexpr uint32_t kAbs = 0x7fff7fffu;
    const uint32_t m2 = max_s16x2(max_s16x2(v.w[0] & kAbs, v.w[1] & kAbs), max_s16x2(v.w[2] & kAbs, v.w[3] & kAbs));
    const uint32_t m = max(m2 & 0xffffu, m2 >> 16);
    if (m < kBf16Inf)
        return m;
    odd = true;
    return odd_eight_top(v.w[0], v.w[1], v.w[2], v.w[3]);
}

__device__ __forceinline__ uint2 eight_convert(const Eight &v, float inverse, bool odd)
{
    if (odd)
        return odd_eight_convert(v.w[0], v.w[1], v.w[2], v.w[3], inverse);
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = to_e4m3x2(bf16_lo(v.w[i]) * inverse, bf16_hi(v.w[i]) * inverse);
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

__device__ __forceinline__ uint32_t element(const __nv_bfloat16 *p)
{
    return __ldg(reinterpret_cast<const uint16_t *>(p));
}

// Elements col .. col+7 of a row of `cols`, one by one, zeros past the end.
__device__ __forceinline__ Eight load_elements(const __nv_bfloat16 *row, uint32_t col, uint32_t cols)
{
    Eight v;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t c = col + 2 * i;
        const uint32_t lo = c < cols ? element(row + c) : 0u;
        const uint32_t hi = c + 1 < cols ? element(row + c + 1) : 0u;
        v.w[i] = lo | (hi << 16);
    }
    return v;
}

// Sixteen lanes load the 128 elements from `col0` of a row, lane i the eight from col0 + 8i (zeros past the row's end).
// VEC: the row starts 16-byte aligned.  Otherwise every lane loads the aligned 16-byte piece its eight begin in, takes the
// next piece from its neighbour (the last lane loads it) and shifts; pieces that reach beyond the row's own elements are
// loaded element by element, so nothing outside the row is read.  All 32 lanes of the warp take part; `mine` = this half
// warp has a row.
template <bool VEC>
__device__ __forceinline__ Eight load_block_row(const __nv_bfloat16 *row, uint32_t col0, uint32_t cols, uint32_t lane16,
                                                bool mine)
{
    const uint32_t col = col0 + lane16 * 8u;
    Eight v{};
    if (VEC) {
        if (mine) {
            if (col + 8 <= cols) {
                const uint4 u = __ldg(reinterpret_cast<const uint4 *>(row + col));
                v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
            } else {
                v = load_elements(row, col, cols);
            }
        }
        return v;
    }
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + col0) & 15u) / 2u;  // elements past an aligned piece
    // piece i holds the elements first + 8i .. of the row, first = col0 - off (it may lie before the row)
    auto piece = [&](uint32_t i) {
        const int64_t c = static_cast<int64_t>(col0) - off + 8 * static_cast<int64_t>(i);
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (c >= 0 && c + 8 <= static_cast<int64_t>(cols)) {
            u = __ldg(reinterpret_cast<const uint4 *>(row + c));
        } else if (c + 8 > 0 && c < static_cast<int64_t>(cols)) {
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                h[j] = (c + j >= 0 && c + j < static_cast<int64_t>(cols)) ? element(row + c + j) : 0u;
            u = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
        }
        return u;
    };
    uint4 a = make_uint4(0u, 0u, 0u, 0u), last = a;
    if (mine) {
        a = piece(lane16);
        if (lane16 == 15u && off != 0u)
            last = piece(16u);
    }
    uint4 b;
    b.x = __shfl_down_sync(0xffffffffu, a.x, 1, 16);
    b.y = __shfl_down_sync(0xffffffffu, a.y, 1, 16);
    b.z = __shfl_down_sync(0xffffffffu, a.z, 1, 16);
    b.w = __shfl_down_sync(0xffffffffu, a.w, 1, 16);
    if (lane16 == 15u)
        b = last;
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (off & 4u) {
#pragma unroll
        for (int i = 0; i < 6; ++i)
            w[i] = w[i + 2];
    }
    if (off & 2u) {
#pragma unroll
        for (int i = 0; i < 5; ++i)
            w[i] = w[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v.w[i] = (off & 1u) ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    return v;
}

// Sixteen lanes store 128 bytes from `col0` of a row of Q, lane i the eight from col0 + 8i (none past the row's end).
// VEC: the row starts 8-byte aligned.  Otherwise each lane stores the two aligned words that end with its bytes, the first
// of them with its neighbour's last bytes; the ends of the run go byte by byte.  All 32 lanes take part.
template <bool VEC>
__device__ __forceinline__ void store_block_row(uint8_t *row, uint32_t col0, uint32_t cols, uint32_t lane16, bool mine, uint2 b)
{
    const uint32_t col = col0 + lane16 * 8u;
    auto bytes = [&](uint32_t from, uint32_t to) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i >= from && i < to)
                row[col + i] = static_cast<uint8_t>((i < 4 ? b.x : b.y) >> (8 * (i & 3u)));
    };
    const bool full = col + 8 <= cols;
    if (VEC) {
        if (mine && full)
            *reinterpret_cast<uint2 *>(row + col) = b;
        else if (mine && col < cols)
            bytes(0u, cols - col);
        return;
    }
    const uint32_t before = __shfl_up_sync(0xffffffffu, b.y, 1, 16);
    if (!mine || col >= cols)
        return;
    if (!full) {
        bytes(0u, cols - col);
        return;
    }
    const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + col) & 3u);
    uint32_t *word = reinterpret_cast<uint32_t *>(row + col - s);
    if (s == 0u || lane16 != 0u)
        word[0] = __funnelshift_l(before, b.x, 8u * s);
    else
        bytes(0u, 4u - s);
    word[1] = __funnelshift_l(b.x, b.y, 8u * s);
    if (s != 0u && (lane16 == 15u || col + 16 > cols))
        bytes(8u - s, 8u);
}

// 1 x 128 blocks: 16 lanes of a warp hold one block, eight elements each; every half warp keeps UNROLL blocks in flight.
template <bool VEC, uint32_t UNROLL>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p)
{
    if (p.pdl) {
        ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t across = (p.cols + kQuantBlock - 1) / kQuantBlock;
    const uint32_t lane16 = threadIdx.x & 15u;
    // Half warp i takes the blocks i, i + step, ... in row order; the row and the block within it are carried along.
    const uint32_t step = gridDim.x * (blockDim.x / 16);
    const uint32_t first = (blockIdx.x * blockDim.x + threadIdx.x) / 16;
    const uint32_t step_rows = step / across, step_blks = step - step_rows * across;
    uint32_t row = first / across, blk = first - row * across;
    // whole warps go round (the shuffles need both halves of one): the warp's first half has the lower block
    for (uint32_t lead = __shfl_sync(0xffffffffu, row, 0); lead < p.rows; lead = __shfl_sync(0xffffffffu, row, 0)) {
        Eight v[UNROLL];
        uint32_t at_row[UNROLL], at_blk[UNROLL];
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            at_row[u] = row;
            at_blk[u] = blk;
            const bool mine = row < p.rows;
            v[u] = load_block_row<VEC>(p.x + static_cast<uint64_t>(mine ? row : 0u) * p.ldx, blk * kQuantBlock, p.cols, lane16, mine);
            row += step_rows;
            blk += step_blks;
            if (blk >= across) {
                blk -= across;
                ++row;
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            const bool mine = at_row[u] < p.rows;
            bool odd = false;
            uint32_t top = eight_top(v[u], odd);
#pragma unroll
            for (uint32_t d = 8; d > 0; d >>= 1)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
            float scale, inverse;
            block_scale(top, scale, inverse);
            store_block_row<VEC>(p.q + static_cast<uint64_t>(mine ? at_row[u] : 0u) * p.ldq, at_blk[u] * kQuantBlock, p.cols, lane16,
                                 mine, eight_convert(v[u], inverse, odd));
            if (mine && lane16 == 0)
                p.scales[static_cast<uint64_t>(at_row[u]) * p.ld_scales + at_blk[u]] = scale;
        }
    }
}

// 128 x 128 blocks: one CTA per block, 16 threads per row, eight rows per thread.
template <bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantParams p)
{
    __shared__ uint32_t warp_top[8];
    if (p.pdl) {
        ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t across = (p.cols + kQuantBlock - 1) / kQuantBlock;
    const uint32_t down = blockIdx.x / across, blk = blockIdx.x - down * across;
    const uint32_t lane16 = threadIdx.x & 15u;
    const uint32_t row0 = down * kQuantBlock + threadIdx.x / 16u;
    Eight v[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = row0 + 16u * i;
        const bool mine = row < p.rows;
        v[i] = load_block_row<VEC>(p.x + static_cast<uint64_t>(mine ? row : 0u) * p.ldx, blk * kQuantBlock, p.cols, lane16, mine);
    }
    bool odd = false;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        top = max(top, eight_top(v[i], odd));
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1)
        top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if ((threadIdx.x & 31u) == 0)
        warp_top[threadIdx.x / 32u] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        top = max(top, warp_top[i]);
    float scale, inverse;
    block_scale(top, scale, inverse);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = row0 + 16u * i;
        const bool mine = row < p.rows;
        store_block_row<VEC>(p.q + static_cast<uint64_t>(mine ? row : 0u) * p.ldq, blk * kQuantBlock, p.cols, lane16, mine,
                             eight_convert(v[i], inverse, odd));
    }
    if (threadIdx.x == 0)
        p.scales[static_cast<uint64_t>(down) * p.ld_scales + blk] = scale;
}

}  // namespace maize
