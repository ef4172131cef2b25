// bf16 -> e4m3 with one power-of-two scale for each block of 1 x 128 or 128 x 128 elements.
//
//     s = 2^p, p = the smallest integer >= -126 with max|x| <= 448 * 2^p  (max over the block's finite elements; 1 if all 0)
//     q = e4m3(x / s), round to nearest even; what is not finite becomes NaN
//
// A power of two makes x / s exact, so the conversion to e4m3 is the only rounding, and it costs no precision: e4m3 keeps
// three mantissa bits at any magnitude down to 2^-6, 14 binades below the largest.
//
// Bound: HBM; 2 bytes read and 1 written per element.  A block's elements stay in registers between the maximum and the
// conversion, so the input is read once.  8192 x 8192: 32.4 us by rows, 32.6 by blocks, 6.2 TB/s.
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

// Sixteen bf16 in eight words: what a lane holds.  Eight lanes hold a row of a block.
struct Sixteen {
    uint32_t w[8];
};
constexpr uint32_t kLaneElements = 16;

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

constexpr uint32_t kBf16Inf = 0x7f80u;

// The sixteen one by one, where one of them is infinite or NaN: the largest finite magnitude, and the conversion with NaN in
// their places (the conversion instruction would saturate infinities).  Out of line: nearly no data comes here.
static __device__ __noinline__ uint32_t odd_top(const Sixteen v)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t lo = v.w[i] & 0x7fffu, hi = (v.w[i] >> 16) & 0x7fffu;
        m = max(m, max(lo < kBf16Inf ? lo : 0u, hi < kBf16Inf ? hi : 0u));
    }
    return m;
}

static __device__ __noinline__ uint4 odd_convert(const Sixteen v, float inverse)
{
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float nan = __uint_as_float(0x7fffffffu);
        h[i] = to_e4m3x2((v.w[i] & 0x7fffu) >= kBf16Inf ? nan : bf16_lo(v.w[i]) * inverse,
                         ((v.w[i] >> 16) & 0x7fffu) >= kBf16Inf ? nan : bf16_hi(v.w[i]) * inverse);
    }
    return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}

// Largest finite magnitude of the sixteen, as bf16 bits (they order like integers); `odd` is set where one is not finite.
__device__ __forceinline__ uint32_t lane_top(const Sixteen &v, bool &odd)
{
    constexpr uint32_t kAbs = 0x7fff7fffu;
    uint32_t m2 = v.w[0] & kAbs;
#pragma unroll
    for (int i = 1; i < 8; ++i)
        m2 = max_s16x2(m2, v.w[i] & kAbs);
    const uint32_t m = max(m2 & 0xffffu, m2 >> 16);
    if (m < kBf16Inf)
        return m;
    odd = true;
    return odd_top(v);
}

__device__ __forceinline__ uint4 lane_convert(const Sixteen &v, float inverse, bool odd)
{
    if (odd)
        return odd_convert(v, inverse);
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        h[i] = to_e4m3x2(bf16_lo(v.w[i]) * inverse, bf16_hi(v.w[i]) * inverse);
    return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}

// Elements c .. c+7 of a row of `cols` as four words; those outside [0, cols) are zeros and not read.  Ordinary loads, here and
// below: the kernel before may still be writing X when this one starts, and the wait for it orders these, but not loads by
// the read-only path.
__device__ __forceinline__ uint4 load_elements(const __nv_bfloat16 *row, int32_t c, int32_t cols)
{
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        h[j] = (c + j >= 0 && c + j < cols) ? *reinterpret_cast<const uint16_t *>(row + c + j) : 0u;
    return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}

// Elements c .. c+7 where row + c is 16-byte aligned: one load where all of them are the row's own, else one by one.
__device__ __forceinline__ uint4 load_piece(const __nv_bfloat16 *row, int32_t c, int32_t cols)
{
    if (c >= 0 && c + 8 <= cols)
        return *reinterpret_cast<const uint4 *>(row + c);
    if (c + 8 > 0 && c < cols)
        return load_elements(row, c, cols);
    return make_uint4(0u, 0u, 0u, 0u);
}

// Eight lanes load the 128 elements from `col0` of a row, lane i the sixteen from col0 + 16i (zeros past the row's end).
// Where the row starts 16-byte aligned, two loads bring them.  Otherwise every lane loads the two aligned 16-byte pieces its
// sixteen begin in (load_pair), gets the next piece from the lane that holds it, or loads it, and shifts (shift_pair);
// nothing outside the row is read.
struct Pair {
    uint4 a, b;
};

// Elements of the row by which the block's first element is past an aligned piece.
__device__ __forceinline__ uint32_t piece_offset(const __nv_bfloat16 *row, uint32_t col0)
{
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + col0) & 15u) / 2u;
}

__device__ __forceinline__ Pair load_pair(const __nv_bfloat16 *row, uint32_t col0, uint32_t cols, uint32_t lane8, uint32_t off, bool mine)
{
    Pair r{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    // the first piece in elements of the row: it may begin before the row
    const int32_t c = static_cast<int32_t>(col0 + lane8 * kLaneElements - off), end = static_cast<int32_t>(cols);
    if (mine) {
        r.a = load_piece(row, c, end);
        r.b = load_piece(row, c + 8, end);
    }
    return r;
}

__device__ __forceinline__ uint4 shfl_down4(const uint4 &v)
{
    return make_uint4(__shfl_down_sync(0xffffffffu, v.x, 1), __shfl_down_sync(0xffffffffu, v.y, 1),
                      __shfl_down_sync(0xffffffffu, v.z, 1), __shfl_down_sync(0xffffffffu, v.w, 1));
}

__device__ __forceinline__ uint4 shfl4(const uint4 &v, int lane)
{
    return make_uint4(__shfl_sync(0xffffffffu, v.x, lane), __shfl_sync(0xffffffffu, v.y, lane), __shfl_sync(0xffffffffu, v.z, lane),
                      __shfl_sync(0xffffffffu, v.w, lane));
}

__device__ __forceinline__ Sixteen shift_pair(const Pair &r, const uint4 &n, uint32_t off)
{
    const uint4 a = r.a, b = r.b;
    uint32_t w[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, n.x, n.y, n.z, n.w};
    if (off & 4u) {
#pragma unroll
        for (int i = 0; i < 10; ++i)
            w[i] = w[i + 2];
    }
    if (off & 2u) {
#pragma unroll
        for (int i = 0; i < 9; ++i)
            w[i] = w[i + 1];
    }
    Sixteen v;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v.w[i] = (off & 1u) ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    return v;
}

__device__ __forceinline__ uint4 shfl_up4(const uint4 &v)
{
    return make_uint4(__shfl_up_sync(0xffffffffu, v.x, 1), __shfl_up_sync(0xffffffffu, v.y, 1), __shfl_up_sync(0xffffffffu, v.z, 1),
                      __shfl_up_sync(0xffffffffu, v.w, 1));
}

// The lane's sixteen bytes b to row + col .. (none past the row's end).  VEC: the row starts 16-byte aligned.  Otherwise a
// lane stores the aligned sixteen bytes that end with its own, the first of them the last of `before`, the sixteen in front
// of its own (`joined`: the row has them and a lane of this warp holds them); the ends of a run go in pieces.  `follows`: a
// lane of this warp holds the next sixteen, if the row has all of them.
template <bool VEC>
__device__ __forceinline__ void store_lane(uint8_t *row, uint32_t col, uint32_t cols, bool mine, bool joined, bool follows,
                                           const uint4 &before, const uint4 &b)
{
    auto bytes = [&](uint32_t count) {  // the first `count`
        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll 1
        for (uint32_t i = 0; i < count; ++i) {
            const uint32_t word = (i & 8u) ? ((i & 4u) ? w[3] : w[2]) : ((i & 4u) ? w[1] : w[0]);
            row[col + i] = static_cast<uint8_t>(word >> (8 * (i & 3u)));
        }
    };
    const bool full = col + 16 <= cols;
    if (VEC) {
        if (mine && full)
            *reinterpret_cast<uint4 *>(row + col) = b;
        else if (mine && col < cols)
            bytes(cols - col);
        return;
    }
    uint32_t w[8] = {before.x, before.y, before.z, before.w, b.x, b.y, b.z, b.w};
    if (!mine || col >= cols)
        return;
    if (!full) {
        // the neighbour's store ends where it ends: these go byte by byte, with its last ones (it has no follower)
        bytes(cols - col);
        return;
    }
    const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + col) & 15u);
    if (s == 0u) {
        *reinterpret_cast<uint4 *>(row + col) = b;
        return;
    }
    if (joined) {
        const uint32_t t = 16u - s;  // bytes of the sixteen before that come first
        if (t & 8u) {
#pragma unroll
            for (int i = 0; i < 6; ++i)
                w[i] = w[i + 2];
        }
        if (t & 4u) {
#pragma unroll
            for (int i = 0; i < 5; ++i)
                w[i] = w[i + 1];
        }
        const uint32_t r = 8u * (t & 3u);
        *reinterpret_cast<uint4 *>(row + col - s) = make_uint4(__funnelshift_r(w[0], w[1], r), __funnelshift_r(w[1], w[2], r),
                                                               __funnelshift_r(w[2], w[3], r), __funnelshift_r(w[3], w[4], r));
    } else {
        // the first 16 - s bytes, up to an aligned address: 1, 2, 4, 8 as the count has them
        uint32_t v[4] = {b.x, b.y, b.z, b.w};
        uint8_t *to = row + col;
        const uint32_t t = 16u - s;
        if (t & 1u) {
            *to = static_cast<uint8_t>(v[0]);
            to += 1;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = __funnelshift_r(v[i], i < 3 ? v[i + 1] : 0u, 8);
        }
        if (t & 2u) {
            *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(v[0]);
            to += 2;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = __funnelshift_r(v[i], i < 3 ? v[i + 1] : 0u, 16);
        }
        if (t & 4u) {
            *reinterpret_cast<uint32_t *>(to) = v[0];
            to += 4;
            v[0] = v[1], v[1] = v[2];
        }
        if (t & 8u)
            *reinterpret_cast<uint2 *>(to) = make_uint2(v[0], v[1]);
    }
    if (!(follows && col + 32 <= cols)) {
        // the last s bytes, from an aligned address: 8, 4, 2, 1.  They are the top of the sixteen: shifted down first.
        uint32_t v[7] = {b.x, b.y, b.z, b.w, 0u, 0u, 0u};
        const uint32_t t = 16u - s;
        if (t & 8u)
            v[0] = v[2], v[1] = v[3], v[2] = 0u, v[3] = 0u;
        if (t & 4u)
            v[0] = v[1], v[1] = v[2], v[2] = v[3], v[3] = 0u;
        const uint32_t r = 8u * (t & 3u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = __funnelshift_r(v[i], v[i + 1], r);
        uint8_t *to = row + col + t;
        if (s & 8u) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(v[0], v[1]);
            to += 8;
            v[0] = v[2], v[1] = v[3];
        }
        if (s & 4u) {
            *reinterpret_cast<uint32_t *>(to) = v[0];
            to += 4;
            v[0] = v[1];
        }
        if (s & 2u) {
            *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(v[0]);
            to += 2;
            v[0] >>= 16;
        }
        if (s & 1u)
            *to = static_cast<uint8_t>(v[0]);
    }
}

// 1 x 128 blocks: eight lanes hold a block, a warp four neighbouring ones at a time and UNROLL times that in a run; only at
// the ends of a run are rows of Q that start anywhere stored in pieces.
template <bool XVEC, bool QVEC, uint32_t UNROLL>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p)
{
    if (p.pdl) {
        ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t across = (p.cols + kQuantBlock - 1) / kQuantBlock;
    const uint32_t lane = threadIdx.x & 31u, lane8 = threadIdx.x & 7u;
    const uint32_t warps = gridDim.x * (blockDim.x / 32), warp = (blockIdx.x * blockDim.x + threadIdx.x) / 32;
    // from one run of this warp to its next, in rows and blocks (a division here, none below)
    const uint32_t step = (warps - 1) * UNROLL * 4;
    const uint32_t step_rows = step / across, step_blks = step - step_rows * across;
    const uint32_t four_rows = 4u / across, four_blks = 4u - four_rows * across;
    const uint64_t first = static_cast<uint64_t>(warp) * UNROLL * 4 + lane / 8u;
    uint32_t row = static_cast<uint32_t>(first / across), blk = static_cast<uint32_t>(first - static_cast<uint64_t>(row) * across);
    auto advance = [&](uint32_t rows, uint32_t blks) {
        row += rows;
        blk += blks;
        if (blk >= across) {
            blk -= across;
            ++row;
        }
    };
    // whole warps go round (the shuffles need every group of one): the warp's first group has the lowest block
    while (__shfl_sync(0xffffffffu, row, 0) < p.rows) {
        Pair raw[UNROLL];
        Sixteen v[UNROLL];
        uint32_t at_row[UNROLL], at_blk[UNROLL], off[UNROLL];
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            at_row[u] = row;
            at_blk[u] = blk;
            const bool mine = row < p.rows;
            const __nv_bfloat16 *x = p.x + static_cast<uint64_t>(mine ? row : 0u) * p.ldx;
            off[u] = XVEC ? 0u : piece_offset(x, blk * kQuantBlock);
            raw[u] = load_pair(x, blk * kQuantBlock, p.cols, lane8, off[u], mine);
            advance(four_rows, four_blks);
        }
        advance(step_rows, step_blks);
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            if (XVEC) {
                v[u] = Sixteen{{raw[u].a.x, raw[u].a.y, raw[u].a.z, raw[u].a.w, raw[u].b.x, raw[u].b.y, raw[u].b.z, raw[u].b.w}};
                continue;
            }
            // the next piece: the lane after holds it, for the last lane the first one of the run's next four blocks
            uint4 n = shfl_down4(raw[u].a);
            if (u + 1 < UNROLL) {
                const uint4 next = shfl4(raw[u + 1].a, 0);
                if (lane == 31u)
                    n = next;
            }
            if (lane8 == 7u && ((u + 1 == UNROLL && lane == 31u) || at_blk[u] + 1 == across)) {
                n = make_uint4(0u, 0u, 0u, 0u);
                if (at_row[u] < p.rows && off[u] != 0u)
                    n = load_piece(p.x + static_cast<uint64_t>(at_row[u]) * p.ldx,
                                   static_cast<int32_t>(at_blk[u] * kQuantBlock + 8u * kLaneElements - off[u]),
                                   static_cast<int32_t>(p.cols));
            }
            v[u] = shift_pair(raw[u], n, off[u]);
        }
        uint4 last = make_uint4(0u, 0u, 0u, 0u);  // lane 31's bytes of the four blocks before
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            const bool mine = at_row[u] < p.rows;
            bool odd = false;
            uint32_t top = lane_top(v[u], odd);
#pragma unroll
            for (uint32_t d = 4; d > 0; d >>= 1)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
            float scale, inverse;
            block_scale(top, scale, inverse);
            const uint4 b = lane_convert(v[u], inverse, odd);
            uint4 before = last;
            if (!QVEC) {
                const uint4 up = shfl_up4(b);
                if (lane != 0u)
                    before = up;
                if (u + 1 < UNROLL)
                    last = shfl4(b, 31);
            }
            store_lane<QVEC>(p.q + static_cast<uint64_t>(mine ? at_row[u] : 0u) * p.ldq, at_blk[u] * kQuantBlock + lane8 * kLaneElements,
                             p.cols, mine, (lane != 0u || u != 0u) && (lane8 != 0u || at_blk[u] != 0u), lane != 31u || u + 1 < UNROLL,
                             before, b);
            if (mine && lane8 == 0)
                p.scales[static_cast<uint64_t>(at_row[u]) * p.ld_scales + at_blk[u]] = scale;
        }
    }
}

// 128 x 128 blocks: one CTA per block, eight threads per row, four rows per thread.
template <bool XVEC, bool QVEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantParams p)
{
    __shared__ uint32_t warp_top[8];
    if (p.pdl) {
        ptx::grid_dependency_launch_dependents();
        ptx::grid_dependency_wait();
    }
    const uint32_t across = (p.cols + kQuantBlock - 1) / kQuantBlock;
    const uint32_t down = blockIdx.x / across, blk = blockIdx.x - down * across;
    const uint32_t lane8 = threadIdx.x & 7u;
    const uint32_t row0 = down * kQuantBlock + threadIdx.x / 8u;
    Pair raw[4];
    Sixteen v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = row0 + 32u * i;
        const bool mine = row < p.rows;
        const __nv_bfloat16 *x = p.x + static_cast<uint64_t>(mine ? row : 0u) * p.ldx;
        raw[i] = load_pair(x, blk * kQuantBlock, p.cols, lane8, XVEC ? 0u : piece_offset(x, blk * kQuantBlock), mine);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (XVEC) {
            v[i] = Sixteen{{raw[i].a.x, raw[i].a.y, raw[i].a.z, raw[i].a.w, raw[i].b.x, raw[i].b.y, raw[i].b.z, raw[i].b.w}};
            continue;
        }
        const uint32_t row = row0 + 32u * i;
        const __nv_bfloat16 *x = p.x + static_cast<uint64_t>(row < p.rows ? row : 0u) * p.ldx;
        const uint32_t off = piece_offset(x, blk * kQuantBlock);
        uint4 n = shfl_down4(raw[i].a);
        if (lane8 == 7u) {
            n = make_uint4(0u, 0u, 0u, 0u);
            if (row < p.rows && off != 0u)
                n = load_piece(x, static_cast<int32_t>(blk * kQuantBlock + 8u * kLaneElements - off), static_cast<int32_t>(p.cols));
        }
        v[i] = shift_pair(raw[i], n, off);
    }
    bool odd = false;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        top = max(top, lane_top(v[i], odd));
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
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = row0 + 32u * i;
        const bool mine = row < p.rows;
        const uint4 b = lane_convert(v[i], inverse, odd);
        store_lane<QVEC>(p.q + static_cast<uint64_t>(mine ? row : 0u) * p.ldq, blk * kQuantBlock + lane8 * kLaneElements, p.cols, mine,
                         lane8 != 0u, lane8 != 7u, QVEC ? b : shfl_up4(b), b);
    }
    if (threadIdx.x == 0)
        p.scales[static_cast<uint64_t>(down) * p.ld_scales + blk] = scale;
}

}  // namespace maize
