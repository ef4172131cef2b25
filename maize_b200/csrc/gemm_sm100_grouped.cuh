// Products of rows that belong to different weight matrices ("experts"): the rows of A are sorted by group, group g
// owns rows offsets[g] .. offsets[g+1]-1, and
//
//     C[r, :] = A[r, :] * W[g]^T   (W[g] stored N x K)      or      C[r, :] = A[r, :] * W[g]   (W[g] stored K x N).
//
// The offsets live on the device, so the host knows neither the sizes of the groups nor the number of tiles: every CTA
// builds the table of tiles itself (build_group_table below) and the persistent pairs deal the tiles out round robin.  (Groups
// with large tiles first, as the weight gradient has them, cost 1 us more at the start and gained nothing: 16 groups of
// 2000 uneven rows, 2048 x 2048, 39 us instead of 37.  What bounds uneven groups is reading W, not the longest pair.)
//
// The WEIGHTS are the M side of the MMA (256 rows of W per CTA pair, 128 per CTA) and the rows of A the N side: an MMA's
// M is fixed but its N is a field of the run-time instruction descriptor, so the ragged end of a group costs its rows
// rounded up to 32 and not a whole tile.  A group of r rows is cut into ceil(r / 256) near-equal tiles.  With the rows
// of A on the M side a group of 300 rows would multiply 512.
//
// What follows from that: the accumulator is C transposed (TMEM lane = column of C, TMEM column = row of C); the epilogue
// trades neighbouring lanes' halves so that a lane has two columns of one row.  These go through shared memory and TMA stores
// where C's rows allow it, else out as 4-byte (2-byte) stores.
//
// Rows of A past the end of a group's tile may be loaded (they belong to the next group); they meet only accumulator
// columns that are never stored, or lie beyond the MMA's N.  W is a stack of matrices in a 3-D tensor map, so rows and
// columns past N and K arrive as zeros and no group's weights meet another's rows.
//
// Bound: tensor pipe where a group has a few hundred rows or more (8 x 2048 rows, 4096 x 4096: 361 us, 1.52 PFLOP/s), HBM
// (reading W) below (32 rows of 16 groups, 4096 x 2048: 37 to 49 us by where the weights lie, 4.9 to 6.3 TB/s).
#pragma once
#include "gemm_common.cuh"

namespace maize {

constexpr uint32_t kGroupedMaxGroups = 1024;
constexpr uint32_t kGroupedTileRows = 256;   // rows of A per tile at most (the MMA's N)
constexpr uint32_t kGroupedTileCols = 256;   // columns of C per tile (the MMA's M over the pair)
constexpr uint32_t kGroupedRowUnit = 32;     // the pair's N is a multiple of 32: 16 rows of A per CTA

struct GroupedParams {
    __nv_bfloat16 *c;
    uint64_t ldc;            // elements
    uint64_t c_stride;       // elements between the matrices of a stacked result (weight gradient)
    const int32_t *offsets;  // groups + 1
    uint32_t groups;
    uint32_t rows;           // rows of A (and of C): the offsets may not exceed it
    uint32_t n, k;
    uint32_t c_pair_ok;      // 1: a column pair (even, odd) of any row of C is 4-byte aligned
    uint32_t c_vec_ok;       // 1: rows of C are 16-byte aligned
    uint32_t c_tma_ok;       // 1: the tensor map of C is valid
    uint32_t c_evict_first;  // 1: TMA stores of C carry an evict-first L2 hint
    uint32_t pdl;
    DeviceStatus *status;
    uint64_t timeout_ns;
};

// Tensor maps of A for tiles of few rows: boxes of 16, 32, 64 and 128 rows of 64 elements.
struct RowMaps {
    CUtensorMap box[4];
};

struct GroupTable {
    uint32_t *offset;  // shared memory: groups + 1 row numbers
    uint32_t *first;   // shared memory: numbers of row tiles before each group of `order`, then the number of all
    uint16_t *order;   // shared memory: the groups with rows; for the weight gradient all groups, those with most rows first

    __device__ __forceinline__ explicit GroupTable(uint8_t *at)
        : offset(reinterpret_cast<uint32_t *>(at)), first(offset + kGroupedMaxGroups + 4),
          order(reinterpret_cast<uint16_t *>(first + kGroupedMaxGroups + 4))
    {
    }
};
constexpr uint32_t kGroupTableBytes = 2 * 4 * (kGroupedMaxGroups + 4) + 2 * kGroupedMaxGroups;
static_assert(kGroupedMaxGroups <= 65536, "groups are listed in 16 bits");

// Whole CTA.  Reads the offsets (into shared memory if `to` is given) and checks them: offsets that do not ascend, or leave
// [0, rows], are reported as MAIZE_ERR_DEVICE_ABORT and the answer is false.
__device__ __forceinline__ bool load_offsets(const GroupedParams &p, uint32_t *to)
{
    bool bad = false;
    for (uint32_t i = threadIdx.x; i <= p.groups; i += blockDim.x) {
        const int32_t o = p.offsets[i];
        const int32_t before = i > 0 ? p.offsets[i - 1] : 0;
        bad |= o < before || o < 0 || static_cast<uint32_t>(o) > p.rows;
        if (to)
            to[i] = static_cast<uint32_t>(o);
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0 && atomicMax(&p.status->code, kStatusDeviceAbort) < kStatusDeviceAbort) {
            p.status->role = 6;
            p.status->cta = static_cast<int>(blockIdx.x);
        }
        return false;
    }
    return true;
}

// Rows of each of the `nt` near-equal tiles of a group: ceil(rows / nt) rounded up to the unit; TILE_ROWS * (nt - 1) < rows
// leaves rows for the last one.
template <uint32_t UNIT>
__device__ __forceinline__ uint32_t rows_per_tile(uint32_t rows, uint32_t nt)
{
    return ((rows + nt - 1) / nt + UNIT - 1) / UNIT * UNIT;
}

// Whole CTA.  Reads the offsets into shared memory, lists the groups that have rows (with 1000 groups and 300 rows, a walk
// over the empty ones took half of the call: 44 us instead of 13) and counts the row tiles before each.  `tiles` = their
// number; false if the offsets are not right.
template <uint32_t TILE_ROWS>
__device__ __forceinline__ bool build_group_table(const GroupedParams &p, const GroupTable &t, uint32_t &tiles)
{
    if (!load_offsets(p, t.offset))
        return false;
    if (threadIdx.x < 32) {
        uint32_t total = 0, listed = 0;
        for (uint32_t base = 0; base < p.groups; base += 32) {
            const uint32_t g = base + threadIdx.x;
            const uint32_t mine = g < p.groups ? (t.offset[g + 1] - t.offset[g] + TILE_ROWS - 1) / TILE_ROWS : 0u;
            const uint32_t with_rows = __ballot_sync(0xffffffffu, mine != 0);
            uint32_t sum = mine;
#pragma unroll
            for (uint32_t d = 1; d < 32; d <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, sum, d);
                if (threadIdx.x >= d)
                    sum += up;
            }
            if (mine != 0) {
                const uint32_t at = listed + __popc(with_rows & ((1u << threadIdx.x) - 1u));
                t.first[at] = total + sum - mine;
                t.order[at] = static_cast<uint16_t>(g);
            }
            listed += __popc(with_rows);
            total += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (threadIdx.x == 0) {
            t.first[listed] = total;
            t.offset[kGroupedMaxGroups + 1] = total;
        }
    }
    __syncthreads();
    tiles = t.offset[kGroupedMaxGroups + 1];
    return true;
}

// One tile: `rows` rows of A from `row0` (group `group`), columns n_blk * 256 .. of C.
struct GroupedTile {
    uint32_t group, n_blk, row0, rows;
    __device__ __forceinline__ uint32_t mma_n() const
    {
        return (rows + kGroupedRowUnit - 1) / kGroupedRowUnit * kGroupedRowUnit;
    }
};

// Tile `t` of the launch; `at` is the role's cursor over the listed groups (tiles come in ascending order).  Within a group the
// row tiles of one block of weights follow each other, so that the weights are read from HBM once.
template <uint32_t UNIT>
__device__ __forceinline__ GroupedTile grouped_tile(uint64_t t, uint32_t n_blocks, const GroupTable &tab, uint32_t &at)
{
    while (t >= static_cast<uint64_t>(tab.first[at + 1]) * n_blocks)
        ++at;
    const uint32_t g = tab.order[at];
    const uint32_t begin = tab.offset[g];
    const uint32_t rows = tab.offset[g + 1] - begin;
    const uint32_t nt = tab.first[at + 1] - tab.first[at];
    const uint32_t local = static_cast<uint32_t>(t - static_cast<uint64_t>(tab.first[at]) * n_blocks);
    const uint32_t tb = local % nt;
    const uint32_t per = rows_per_tile<UNIT>(rows, nt);
    GroupedTile r;
    r.group = g;
    r.n_blk = local / nt;
    r.row0 = begin + tb * per;
    r.rows = min(per, rows - tb * per);
    return r;
}

// The grouped kernel has eight epilogue warps, two for each quarter of the lanes: they take the 32-row chunks of a tile in
// turn.  Two warps with neighbouring quarters share a staging buffer of 32 rows x 64 columns.
constexpr uint32_t kGroupedEpilogueWarps = 8;
constexpr uint32_t kGroupedThreads = 64 + 32 * kGroupedEpilogueWarps;

template <uint32_t STAGES>
struct GroupedSmemLayout {
    static constexpr uint32_t kWBytes = kBlockM * kBlockK * 2;                  // this CTA's 128 rows of W, one k-block
    static constexpr uint32_t kABytes = (kGroupedTileRows / 2) * kBlockK * 2;   // this CTA's half of the rows of A
    static constexpr uint32_t kStageBytes = kWBytes + kABytes;
    static constexpr uint32_t kStagingOffset = STAGES * kStageBytes;
    static constexpr uint32_t kBarOffset = kStagingOffset + kGroupedEpilogueWarps / 2 * kTmaStoreBufBytes;
    static constexpr uint32_t kNumBars = 2 * STAGES + 4;
    static constexpr uint32_t kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr uint32_t kAbortOffset = kTmemSlotOffset + 4;
    static constexpr uint32_t kTableOffset = (kAbortOffset + 4 + 15) / 16 * 16;
    static constexpr uint32_t kUsedBytes = kTableOffset + kGroupTableBytes;
    static constexpr uint32_t kDynamicBytes = kUsedBytes + 1024;
    static_assert(kDynamicBytes <= 232448, "exceeds 227 KiB of shared memory per CTA");
    static_assert(kDynamicBytes > 116224, "two CTAs could share an SM and contend for TMEM");
};

// Stores 32 rows (TMEM columns) x 32 columns of C (lanes) held by a warp.  `row0` = first row, `valid` = rows of the
// chunk that belong to the tile (warp-uniform), `col` = this lane's column of C.
__device__ __forceinline__ void store_transposed_chunk(const GroupedParams &p, uint32_t row0, uint32_t valid,
                                                       uint32_t col, uint32_t lane, const uint32_t (&acc)[32])
{
    if (p.c_pair_ok) {
        // Rows j and j+1 of a lane are packed into one word; the even lane of a pair keeps row j of both lanes, the
        // odd lane row j+1: each lane then holds two neighbouring columns of one row.
        const bool odd = (lane & 1u) != 0u;
        const uint32_t col2 = col & ~1u;
        __nv_bfloat16 *base = p.c + static_cast<uint64_t>(row0 + (odd ? 1u : 0u)) * p.ldc + col2;
        const bool both = col2 + 1 < p.n, first = col2 < p.n;
#pragma unroll
        for (uint32_t j = 0; j < 32; j += 2) {
            const uint32_t mine = ptx::pack_bf16x2(acc[j], acc[j + 1]);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
            const uint32_t word = odd ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);
            if (j + (odd ? 1u : 0u) < valid) {
                __nv_bfloat16 *dst = base + static_cast<uint64_t>(j) * p.ldc;
                if (both)
                    *reinterpret_cast<uint32_t *>(dst) = word;
                else if (first)
                    *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(word);
            }
        }
        return;
    }
    if (col >= p.n)
        return;
    __nv_bfloat16 *dst = p.c + static_cast<uint64_t>(row0) * p.ldc + col;
#pragma unroll
    for (uint32_t j = 0; j < 32; ++j)
        if (j < valid)
            dst[static_cast<uint64_t>(j) * p.ldc] = __float2bfloat16_rn(__uint_as_float(acc[j]));
}

// The same for C that TMA can store: two warps write their 32 columns each as rows of 64 into a shared buffer (16-byte chunk
// j of row r at j ^ (r & 7)); all 32 rows of a whole chunk leave as one TMA store of 128-byte rows, those of a chunk that the
// group's end cuts are stored row by row.  `half` = which of the two warps, `barrier` = the pair's barrier.
__device__ __forceinline__ void store_transposed_chunk_tma(const GroupedParams &p, const CUtensorMap *tma_c, uint32_t stage_u32,
                                                           uint32_t barrier, uint32_t half, uint32_t row0, uint32_t valid,
                                                           uint32_t col0, uint32_t lane, const uint32_t (&acc)[32])
{
    if (half == 0 && lane == 0)
        ptx::bulk_wait_group_read<0>();  // the buffer's last store has read it
    ptx::named_barrier(barrier, 64);
    const bool odd = (lane & 1u) != 0u;
    const uint32_t chunk = half * 4u + (lane >> 3), at = ((lane >> 1) & 3u) * 4u;
#pragma unroll
    for (uint32_t j = 0; j < 32; j += 2) {
        const uint32_t mine = ptx::pack_bf16x2(acc[j], acc[j + 1]);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
        const uint32_t word = odd ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);
        const uint32_t r = j + (odd ? 1u : 0u);
        ptx::st_shared_u32(stage_u32 + r * 128u + ((chunk ^ (r & 7u)) << 4) + at, word);
    }
    ptx::fence_proxy_async_shared();
    ptx::named_barrier(barrier, 64);
    if (valid == 32u) {
        if (half == 0 && lane == 0) {
            ptx::tma_store_2d(tma_c, stage_u32, static_cast<int32_t>(col0), static_cast<int32_t>(row0));
            ptx::bulk_commit_group();
        }
    } else {
        const uint32_t col = col0 + lane * 2u;
        for (uint32_t r = half; r < valid; r += 2) {
            const uint32_t word = ptx::ld_shared_u32(stage_u32 + r * 128u + (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u);
            if (col < p.n)  // N is even
                *reinterpret_cast<uint32_t *>(p.c + static_cast<uint64_t>(row0 + r) * p.ldc + col) = word;
        }
    }
    __syncwarp();
}

// W_KN: the weights are stored K x N; this CTA's 128 columns are two boxes of {64 columns, 64 k-rows} per k-block, read
// by the MMA as an MN-major operand.
template <bool W_KN, uint32_t STAGES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGroupedThreads, 1)
gemm_bf16_sm100_grouped(const __grid_constant__ RowMaps tma_a, const __grid_constant__ CUtensorMap tma_w,
                        const __grid_constant__ CUtensorMap tma_c, const GroupedParams p)
{
    using L = GroupedSmemLayout<STAGES>;
    constexpr uint32_t kTmemCols = 2 * kGroupedTileRows;  // two accumulator buffers of 256 columns
    constexpr uint32_t kChunkBytes = kBlockK * 128;       // one 64-column chunk of a K x N tile: 64 k-rows x 128 B

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemSlotOffset);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbortOffset);
    const GroupTable tab(smem_gen + L::kTableOffset);

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t cta_rank = ptx::cluster_cta_rank();
    const uint32_t pair = blockIdx.x >> 1;
    const uint32_t num_pairs = gridDim.x >> 1;
    const uint32_t num_steps = (p.k + kBlockK - 1) / kBlockK;
    const uint32_t n_blocks = (p.n + kGroupedTileCols - 1) / kGroupedTileCols;
    const WaitCtl ctl{abort_flag, p.status, p.timeout_ns};

    if (threadIdx.x == 0) {
        ptx::prefetch_tensormap(&tma_w);
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);   // the leader's producer; bytes of both CTAs
            ptx::mbar_init(empty_bar(s), 1);  // one tcgen05.commit of the leader
        }
        for (uint32_t b = 0; b < 2; ++b) {
            ptx::mbar_init(acc_full_bar(b), 1);
            ptx::mbar_init(acc_empty_bar(b), 2 * kGroupedEpilogueWarps);
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
    // both CTAs of a pair read the same offsets and come to the same tiles
    uint32_t row_tiles = 0;
    build_group_table<kGroupedTileRows>(p, tab, row_tiles);
    const uint64_t num_tiles = static_cast<uint64_t>(row_tiles) * n_blocks;

    bool role_ok = true;
    if (warp == 0) {
        // ------------------------------------------------------- TMA producer --
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, g = 0;
            bool ok = true;
            for (uint64_t t = pair; ok && t < num_tiles; t += num_pairs) {
                const GroupedTile tile = grouped_tile<kGroupedRowUnit>(t, n_blocks, tab, g);
                const uint32_t half = tile.mma_n() / 2;  // rows of A this CTA brings in
                const uint32_t box = half <= 16 ? 0u : (half <= 32 ? 1u : (half <= 64 ? 2u : 3u));
                const uint32_t a_bytes = (16u << box) * (kBlockK * 2);
                const int32_t r0 = static_cast<int32_t>(tile.row0 + cta_rank * half);
                const int32_t n0 = static_cast<int32_t>(tile.n_blk * kGroupedTileCols + cta_rank * kBlockM);
                for (uint32_t step = 0; step < num_steps; ++step) {
                    ok = wait_bounded<true>(empty_bar(stage), phase ^ 1u, ctl, 1);
                    if (!ok)
                        break;
                    const uint32_t sw = smem_base + stage * L::kStageBytes;
                    const uint32_t sa = sw + L::kWBytes;
                    const uint32_t leader_full = ptx::mapa_shared(full_bar(stage), 0);
                    const int32_t kx = static_cast<int32_t>(step * kBlockK);
                    if (cta_rank == 0)
                        ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * (L::kWBytes + a_bytes));
                    if constexpr (W_KN) {
#pragma unroll
                        for (uint32_t j = 0; j < 2; ++j)
                            ptx::tma_load_3d_pair(sw + j * kChunkBytes, &tma_w, leader_full,
                                                  n0 + static_cast<int32_t>(64u * j), kx, static_cast<int32_t>(tile.group));
                    } else {
                        ptx::tma_load_3d_pair(sw, &tma_w, leader_full, kx, n0, static_cast<int32_t>(tile.group));
                    }
                    ptx::tma_load_2d_pair(sa, &tma_a.box[box], leader_full, kx, r0);
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
        // ------------------------------------------- MMA issuer (leader only) --
        if (lane == 0 && cta_rank == 0) {
            uint32_t stage = 0, phase = 0, g = 0;
            uint32_t acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint64_t t = pair; ok && t < num_tiles; t += num_pairs) {
                const GroupedTile tile = grouped_tile<kGroupedRowUnit>(t, n_blocks, tab, g);
                const uint32_t idesc = ptx::make_instr_desc_bf16(2 * kBlockM, tile.mma_n(), false, W_KN);
                ok = wait_bounded<true>(acc_empty_bar(acc), acc_phase ^ 1u, ctl, 2);
                if (!ok)
                    break;
                ptx::tcgen05_fence_after();
                const uint32_t tmem_d = tmem_base + acc * kGroupedTileRows;
                for (uint32_t step = 0; step < num_steps; ++step) {
                    ok = wait_bounded<true>(full_bar(stage), phase, ctl, 2);
                    if (!ok)
                        break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sw = smem_base + stage * L::kStageBytes;
                    const uint64_t dw = W_KN ? ptx::make_smem_desc_sw128_mn(sw, kChunkBytes) : ptx::make_smem_desc_sw128(sw);
                    const uint64_t da = ptx::make_smem_desc_sw128(sw + L::kWBytes);
                    constexpr uint32_t kStepW = W_KN ? 128u : 2u;  // +2048 B or +32 B per 16-wide K step
#pragma unroll
                    for (uint32_t k = 0; k < kBlockK / kUmmaK; ++k)
                        ptx::mma_bf16_2cta(tmem_d, dw + kStepW * k, da + 2u * k, idesc, (step | k) != 0u ? 1u : 0u);
                    ptx::mma_commit_2cta_mask(empty_bar(stage), 3);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok)
                    break;
                ptx::mma_commit_2cta_mask(acc_full_bar(acc), 3);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            role_ok = ok;
        }
        __syncwarp();
    } else {
        // ----------------------------------------------------------- epilogue --
        const uint32_t quarter = warp & 3u, turn = (warp - 2u) >> 2;  // this warp takes every other chunk of 32 rows
        const uint32_t share = turn * 2u + (quarter >> 1);               // buffer and barrier of the two warps side by side
        const uint32_t stage_u32 = smem_base + L::kStagingOffset + share * kTmaStoreBufBytes;
        uint32_t acc = 0, acc_phase = 0, g = 0;
        bool ok = true;
        for (uint64_t t = pair; ok && t < num_tiles; t += num_pairs) {
            const GroupedTile tile = grouped_tile<kGroupedRowUnit>(t, n_blocks, tab, g);
            ok = wait_bounded<true>(acc_full_bar(acc), acc_phase, ctl, 3);
            // both warps of a buffer go on or both give up: neither may wait at their barrier for one that has left
            ok = ptx::named_barrier_and(1u + share, 64, ok);
            if (!ok)
                break;
            ptx::tcgen05_fence_after();
            const uint32_t taddr = tmem_base + acc * kGroupedTileRows + ((quarter * 32u) << 16);
            const uint32_t pair_col = tile.n_blk * kGroupedTileCols + cta_rank * kBlockM + (quarter >> 1) * 64u;
            const uint32_t warp_col = pair_col + (quarter & 1u) * 32u;
            // The accumulator goes back as soon as it is in registers, without a release: the loads are complete, and a release
            // at cluster scope would wait for the warp's stores.
            auto hand_back = [&] {
                ptx::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive_cluster_addr_relaxed(ptx::mapa_shared(acc_empty_bar(acc), 0));
            };
            if (pair_col < p.n && turn * 32u < tile.rows) {
#pragma unroll 1
                for (uint32_t r = turn * 32u; r < tile.rows; r += 64) {
                    uint32_t v[32];
                    ptx::tmem_ld_32x32b_x32(taddr + r, v);
                    ptx::tmem_ld_wait();
                    if (r + 64 >= tile.rows)
                        hand_back();
                    const uint32_t valid = min(32u, tile.rows - r);
                    if (p.c_tma_ok)
                        store_transposed_chunk_tma(p, &tma_c, stage_u32, 1u + share, quarter & 1u, tile.row0 + r, valid, pair_col, lane, v);
                    else if (warp_col < p.n)
                        store_transposed_chunk(p, tile.row0 + r, valid, warp_col + lane, lane, v);
                    __syncwarp();
                }
            } else {
                hand_back();
            }
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        if (p.c_tma_ok)
            tma_store_drain(lane);
        role_ok = ok;
    }
    if (!role_ok) {
        // tell the peer CTA too, so that its roles stop waiting on us
        ptx::st_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(const_cast<int *>(abort_flag)), cta_rank ^ 1u), 1u);
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
        ptx::tmem_dealloc_2cta(tmem_base, kTmemCols);
    }
}

// C rows [offsets[0], offsets[groups]) = 0: the empty sum (K == 0).
static __global__ void __launch_bounds__(256) grouped_zero_rows_kernel(const GroupedParams p)
{
    if (!load_offsets(p, nullptr))
        return;
    const int32_t begin = p.offsets[0], end = p.offsets[p.groups];
    const uint64_t total = static_cast<uint64_t>(end - begin) * p.n;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += stride)
        p.c[(static_cast<uint64_t>(begin) + i / p.n) * p.ldc + i % p.n] = __float2bfloat16_rn(0.0f);
}

}  // namespace maize
