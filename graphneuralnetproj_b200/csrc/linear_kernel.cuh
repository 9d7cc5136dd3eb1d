// Linear layers on dense weights of fewer bytes or of many experts: C[n][m] = sum_k B[n][k] * A[m][k], token-major as
// the eleven-argument SpMM (third_party/ft.patch:2822-2846), with A and B
//   - e4m3 codes with an fp32 scale per 128 x 128 block of A and per token and 128 features of B, or
//   - fp16 / bf16,
// and either one matrix A or one per group of consecutive tokens (experts; group borders are read on the device).
//
// A block takes 128 rows of A as the M side of tcgen05.mma and up to 128 tokens as its N side (N is a run-time field of
// the instruction descriptor, so a group's last few tokens cost no more than they must), because weights are what there
// is always plenty of: one token still fills the tensor core's 128 lanes and streams A at full rate.  A k-block is 128
// bytes of K (64 halves or 128 codes, i.e. one scale block), the width of a 128-byte-swizzled TMA box; a ring stage
// holds a step of two k-blocks, because the MMA lane's waits and commits cost a few hundred cycles per stage.
//
// fp16 / bf16 accumulate the whole K range in TMEM.  With scales every k-block is a product of its own: the MMA warp
// fills one half of TMEM with the products of a group of one to four steps (as many as fit side by side), and the
// epilogue warps add them to fp32 registers, each column times (token's scale) * (block's scale), while the tensor core
// fills the other half.  One hand-over per group, not per step: with a wait for the product and another for the scales
// in every step, the few hundred instructions of the epilogue warps around them took 1.4 us per step, twice what the
// 32 KB of a step take to arrive (36864 x 9216, 16 tokens: 104 us, against 70 without the second wait).
//
// What bounds it: memory.  A block has six stages of 36 KB on their way at 16 tokens; 36864 x 9216 in 8 bits and 16 tokens take
// 57 us (341 MB, 0.91 of the measured copy bandwidth), 64 experts of 2048 x 4096 in bf16 and 96 tokens 114 us (0.97).  A launch
// has about 5 us that do not depend on the size (first loads, last tile's way out), which is what a small layer costs.
//
// MMAs, commits and TMA loads are issued by an elected lane in code that is uniform for the compiler (values that come out of
// shared memory pass through linear_uniform): under `lane == 0` four MMAs and two commits took 520 cycles, now 170.
//
// A launch starts before its predecessor in the stream has finished, which may be what writes the group borders and the scales:
// they are read through L2 (__ldcg), never through the non-coherent path, whose data must not change while a kernel runs.
//
// Roles: warp 0 TMA, warp 1 MMA issue and TMEM, warp 2 scales, warps 4..11 epilogue (warp % 4 = quarter of the TMEM
// lanes, warp / 4 - 1 = every other chunk of columns).  Every wait is bounded; a block that gives up records it.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "linear_plan.h"
#include "ptx_sm100.cuh"

namespace spmm_b200 {

__device__ int g_linear_status;  // 1 after a bounded wait has given up

constexpr int kLinearThreads   = 384;
constexpr int kLinearMaxStages = 12;
constexpr int kLinearMaxGroups = 1024;
constexpr int kLinearRows      = 128;                // lanes of a block's tile
constexpr int kLinearBoxBytes  = kLinearRows * 128;  // its operand, one k-block
constexpr int kStepBlocks      = 2;  // k-blocks per ring stage
constexpr int kGroupBlocks     = 8;  // k-blocks of a group at most
constexpr int kGroupScales     = 256;  // scales of a group: k-blocks x columns
constexpr int kEpilogueTeams   = 8;  // epilogue warps
constexpr int kLinearBand      = 8;
constexpr int kPieceCounters   = 4096;  // arrival counters at the head of a workspace
constexpr int kLinearFixedSmem = 1024 /* alignment */ + 512 /* barriers */;

struct LinearParams {
    CUtensorMap  a_map, b_map;  // bytes: (K bytes, rows, groups)
    const float* a_scales;      // [groups][ceil(M / 128)][kb]
    const float* b_scales;      // [kb][N]
    void*        C;
    const int*   offsets;  // [groups + 1], or null: one group of all N tokens
    unsigned*    counters;
    float*       slots;
    int          groups, m, n;
    int          kb;        // k-blocks
    int          steps;     // pairs of them
    int          nt;        // tokens per tile at most
    int          b_box;     // tokens per TMA box
    int          stages;
    int          bf16;      // C (and 16-bit operands) are bf16, not fp16
    int          wide_c;    // C takes 16-byte stores: aligned, M a multiple of 8
    LinearCutting cutting;
};

// Which part of the layer a tile is.
struct LinearTile {
    int group, m0, row0, rows;  // first row of A, first token, tokens
};

// One element of C, rounded once.
__device__ __forceinline__ void linear_store(const LinearParams& p, size_t at, float v)
{
    if (p.bf16)
        static_cast<__nv_bfloat16*>(p.C)[at] = __float2bfloat16_rn(v);
    else
        static_cast<half*>(p.C)[at] = __float2half_rn(v);
}

// Two of them.
__device__ __forceinline__ uint32_t linear_pair_of(float lo, float hi, int bf16)
{
    uint32_t out;
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        out                    = *reinterpret_cast<const uint32_t*>(&h);
    }
    else {
        const __half2 h = __floats2half2_rn(lo, hi);
        out             = *reinterpret_cast<const uint32_t*>(&h);
    }
    return out;
}

// Stores CH columns (tokens `col` .. of the tile) of accumulators whose lanes are rows of A; all lanes of a warp, `m` this
// lane's row.  Four neighbouring lanes exchange their values for four tokens, so that each stores eight bytes of one token: one
// store instruction for four tokens instead of one for each (2048 x 9472 x 1024 in fp16 spent half of its 43 us on them).
template<int CH>
__device__ __forceinline__ void linear_store_columns(const LinearParams& p, const LinearTile& t, int m, int col, const float* v)
{
    if (!p.wide_c) {
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (m < p.m && col + j < t.rows)
                linear_store(p, static_cast<size_t>(t.row0 + col + j) * p.m + m, v[j]);
        return;
    }
    const int lane = m & 3, first = m - lane;  // rows of a tile start at a multiple of 128
    uint16_t* to   = static_cast<uint16_t*>(p.C) + static_cast<size_t>(t.row0 + col + lane) * p.m + first;
#pragma unroll
    for (int j = 0; j < CH; j += 4) {
        if (col + j >= t.rows)
            break;
        const uint32_t w0 = linear_pair_of(v[j], v[j + 1], p.bf16), w1 = linear_pair_of(v[j + 2], v[j + 3], p.bf16);
        const uint32_t x0 = __shfl_xor_sync(0xffffffffu, w0, 1), x1 = __shfl_xor_sync(0xffffffffu, w1, 1);
        // even lanes: tokens 0 and 2 of their row and the next; odd lanes: tokens 1 and 3 of the row before and theirs
        const uint32_t a0 = (lane & 1) ? __byte_perm(x0, w0, 0x7632) : __byte_perm(w0, x0, 0x5410);
        const uint32_t a1 = (lane & 1) ? __byte_perm(x1, w1, 0x7632) : __byte_perm(w1, x1, 0x5410);
        const uint32_t got = __shfl_xor_sync(0xffffffffu, (lane & 2) ? a0 : a1, 2);
        if (first < p.m && col + j + lane < t.rows)
            *reinterpret_cast<uint2*>(to + static_cast<size_t>(j) * p.m) = (lane & 2) ? make_uint2(got, a1) : make_uint2(a0, got);
    }
}

// The groups, as every role of a block needs them (in shared memory).
struct LinearTable {
    int* end;    // tiles of the groups up to and including this one
    int* row;    // first token
    int* rows;   // tokens
    int* group;  // which group this is
};
constexpr int kLinearTableWords = 4;  // per group
constexpr int kLinearSortGroups = 256;

// Parts of `by` that cover `count`: not negative, and up to INT_MAX, where a sum of the two no longer fits an int.
__device__ __forceinline__ int linear_cover(int count, int by)
{
    return static_cast<int>((static_cast<unsigned>(count) + static_cast<unsigned>(by) - 1u) / static_cast<unsigned>(by));
}

// Tokens per tile of a group: the tiles of a group are as wide as one another, in steps of `granule` columns.
__device__ __forceinline__ int linear_tile_rows(int rows, int tile_tokens, int granule)
{
    const int tiles = linear_cover(rows, tile_tokens);
    return tiles == 0 ? 0 : linear_cover(linear_cover(rows, tiles), granule) * granule;
}

// Fills the table; all threads of the block, with block barriers.  Borders are clamped to the tokens there are, so that a
// corrupt table cannot lead outside.  Tiles are up to `tile_tokens` tokens x one of `tiles_m` blocks of rows of A.
// sort: groups with wider tiles first.  Whole tiles are dealt to the blocks in turn, so that blocks get tiles of about the same
// width only if neighbours in the list have it (16 groups of 124 to 2220 tokens: 542 -> 476 us with equal tiles and sorting).
template<bool SORT>
__device__ __forceinline__ void
linear_build_table(const LinearParams& p, const LinearTable& table, int* warp_sums, int tile_tokens, int granule, int tiles_m)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per  = (p.groups + kLinearThreads - 1) / kLinearThreads;
    const int e0   = min(static_cast<int>(threadIdx.x) * per, p.groups), e1 = min(e0 + per, p.groups);
    for (int e = e0; e < e1; e++) {
        int from = 0, rows = p.n;
        if (p.offsets) {
            from = min(max(__ldcg(p.offsets + e), 0), p.n);
            rows = max(min(max(__ldcg(p.offsets + e + 1), 0), p.n) - from, 0);
        }
        table.row[e]   = from;
        table.rows[e]  = rows;
        table.group[e] = e;
    }
    if (SORT && p.groups > 1 && p.groups <= kLinearSortGroups) {  // at most one group per thread
        __syncthreads();
        int from = 0, rows = 0, rank = 0;
        if (e0 < e1) {
            from            = table.row[e0];
            rows            = table.rows[e0];
            const int width = linear_tile_rows(rows, tile_tokens, granule);
            for (int j = 0; j < p.groups; j++) {
                const int other = linear_tile_rows(table.rows[j], tile_tokens, granule);
                rank += other > width || (other == width && j < e0);
            }
        }
        __syncthreads();
        if (e0 < e1) {
            table.row[rank]   = from;
            table.rows[rank]  = rows;
            table.group[rank] = e0;
        }
        __syncthreads();
    }
    int sum = 0;
    for (int e = e0; e < e1; e++) {
        sum += linear_cover(table.rows[e], tile_tokens) * tiles_m;
        table.end[e] = sum;
    }
    int before = sum;  // becomes the total of the threads before this one
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d)
            before += up;
    }
    if (lane == 31)
        warp_sums[warp] = before;
    before -= sum;
    __syncthreads();
    for (int w = 0; w < warp; w++)
        before += warp_sums[w];
    for (int e = e0; e < e1; e++)
        table.end[e] += before;
    __syncthreads();
}

// Which part of the layer a tile is: `block_rows` rows of A and up to `tile_tokens` tokens.  Tiles that run at the same time
// should share operands in L2: tokens are taken in bands of kLinearBand tiles, in a band a block of rows of A after the other.
__device__ __forceinline__ LinearTile
linear_locate(const LinearParams& p, const LinearTable& table, int tile, int tile_tokens, int granule, int block_rows, int tiles_m)
{
    int lo = 0, hi = p.groups - 1;  // the first group whose running total is above `tile`
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (table.end[mid] > tile)
            hi = mid;
        else
            lo = mid + 1;
    }
    LinearTile t;
    const int  rows = table.rows[lo], tiles_n = linear_cover(rows, tile_tokens);
    const int  width = linear_tile_rows(rows, tile_tokens, granule);
    const int  i    = tile - (lo > 0 ? table.end[lo - 1] : 0);
    const int  band = i / (kLinearBand * tiles_m), wide = min(kLinearBand, tiles_n - band * kLinearBand);
    const int  rest = i - band * kLinearBand * tiles_m;
    t.group = table.group[lo];
    t.m0    = rest / wide * block_rows;
    t.row0  = (band * kLinearBand + rest % wide) * width;
    t.rows  = min(width, rows - t.row0);
    t.row0 += table.row[lo];
    return t;
}

// The value of lane 0, known to the compiler to be the same in all lanes.
__device__ __forceinline__ int linear_uniform(int v)
{
    return __shfl_sync(0xffffffffu, v, 0);
}

// Segments and tiles for the warps that issue MMAs and TMA loads (see ptx::elect_one).
__device__ __forceinline__ LinearSegment linear_uniform(LinearSegment s)
{
    s.tile = linear_uniform(s.tile);
    s.kb0  = linear_uniform(s.kb0);
    s.kb1  = linear_uniform(s.kb1);
    return s;
}
__device__ __forceinline__ LinearTile linear_uniform(LinearTile t)
{
    t.group = linear_uniform(t.group);
    t.m0    = linear_uniform(t.m0);
    t.row0  = linear_uniform(t.row0);
    t.rows  = linear_uniform(t.rows);
    return t;
}

// Steps whose products fit side by side into 256 TMEM columns, and the columns of each.
SPMM_B200_HD int linear_group_steps(int nt)
{
    return nt <= 32 ? 4 : (nt <= 64 ? 2 : 1);
}

// A bounded wait of a whole warp, with the same answer for all of its lanes: warp-wide instructions follow, and a lane that gave
// up while the others saw the phase complete would leave them waiting for it.  The phase cannot pass before all lanes have seen it,
// since the next one needs this warp.  Parked at once: here most waits are long, and the polling of ten warps slows the
// others down (64 experts of 2048 x 4096 in bf16: 130 us with 64 polls before parking, 121 without).
__device__ __forceinline__ bool linear_wait(uint32_t bar, uint32_t parity, volatile int* abort_word, uint64_t limit_ns = ptx::kWaitLimitNs)
{
    uint64_t start = 0;
#pragma unroll 1
    for (uint32_t polls = 0;; polls++) {
        if (__all_sync(0xffffffffu, ptx::mbar_try_wait_suspend(bar, parity, ptx::kSuspendNs)))
            return true;
        bool give_up = *abort_word != 0;
        if ((polls & 255u) == 0) {
            const uint64_t now = ptx::global_timer_ns();
            if (start == 0)
                start = now;
            else if (now - start > limit_ns) {
                *abort_word = 1;
                give_up     = true;
            }
        }
        if (__any_sync(0xffffffffu, give_up))
            return false;
    }
}

constexpr uint64_t kDrainNs = 10000000ull;  // an abandoned block waits so long at most for each copy or product under way

template<bool EIGHT>
__global__ void __launch_bounds__(kLinearThreads, 1)
linear_kernel(const __grid_constant__ LinearParams p)
{
    constexpr int NMAX = 128;             // columns of a tile at most
    constexpr int BUFS = 2;               // halves of TMEM
    constexpr int CH   = 16;              // columns per chunk
    constexpr int NCH  = NMAX / (2 * CH); // chunks per epilogue warp

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base   = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t*       smem        = smem_raw + (smem_base - ptx::smem_addr(smem_raw));
    const uint32_t part_bytes  = p.nt * 128u;  // B's part of a k-block
    const uint32_t stage_bytes = kStepBlocks * (kLinearBoxBytes + part_bytes);
    const int      group_steps = linear_group_steps(p.nt);
    const int      acc_shift   = p.nt <= 32 ? 5 : (p.nt <= 64 ? 6 : 7);
    const int      acc_width   = 1 << acc_shift;  // TMEM columns of a product: group_steps * kStepBlocks * acc_width = 256
    const uint32_t scale_off   = p.stages * stage_bytes;
    const uint32_t bar_off     = scale_off + (EIGHT ? BUFS * kGroupScales * 4u : 0u);
    const uint32_t bar_base    = smem_base + bar_off;
    float* const   scale_ring  = reinterpret_cast<float*>(smem + scale_off);
    auto full       = [&](int s) { return bar_base + 8u * s; };
    auto empty      = [&](int s) { return bar_base + 8u * (kLinearMaxStages + s); };
    auto acc_full   = [&](int b) { return bar_base + 8u * (2 * kLinearMaxStages + b); };
    auto acc_free   = [&](int b) { return bar_base + 8u * (2 * kLinearMaxStages + BUFS + b); };
    const uint32_t     drained = bar_base + 8u * (2 * kLinearMaxStages + 2 * BUFS);
    constexpr uint32_t kWords  = 8u * (2 * kLinearMaxStages + 2 * BUFS + 1);
    static_assert(kWords + 64 <= 512, "barrier block");
    volatile uint32_t* tmem_slot  = reinterpret_cast<volatile uint32_t*>(smem + bar_off + kWords);
    volatile int*      abort_word = reinterpret_cast<volatile int*>(smem + bar_off + kWords + 4);
    int* const         warp_sums  = reinterpret_cast<int*>(smem + bar_off + kWords + 8);  // 12 words
    int* const         groups_at  = reinterpret_cast<int*>(smem + bar_off + 512);
    const LinearTable  table{groups_at, groups_at + p.groups, groups_at + 2 * p.groups, groups_at + 3 * p.groups};

    const int warp = linear_uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kLinearMaxStages; s++) {
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), 1);
        }
        for (int b = 0; b < BUFS; b++) {
            ptx::mbar_init(acc_full(b), EIGHT ? 2 : 1);  // the products, and the scales
            ptx::mbar_init(acc_free(b), kEpilogueTeams);
        }
        ptx::mbar_init(drained, 1);
        *abort_word = 0;
        ptx::mbar_init_fence();
    }
    if (warp == 1) {
        ptx::tmem_alloc(bar_base + kWords, 512);
        ptx::tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        ptx::prefetch_tensor_map(&p.a_map);
        ptx::prefetch_tensor_map(&p.b_map);
    }
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();

    const int tiles_m = (p.m - 1) / kLinearRows + 1;
    ptx::tc_fence_before_sync();
    if (p.offsets == nullptr) {
        // One group: the TMA warp, which set up the barriers, need not wait for the others to start the first loads.
        if (threadIdx.x == 0) {
            table.row[0]   = 0;
            table.rows[0]  = p.n;
            table.group[0] = 0;
            table.end[0]   = linear_cover(p.n, p.nt) * tiles_m;
        }
        __syncwarp();
        if (warp == 0)
            ptx::named_arrive(1, kLinearThreads);
        else
            ptx::named_sync(1, kLinearThreads);
    }
    else
        linear_build_table<false>(p, table, warp_sums, p.nt, 16, tiles_m);
    ptx::tc_fence_after_sync();
    const uint32_t        tmem_base = warp == 0 ? 0 : linear_uniform(static_cast<int>(*tmem_slot));
    const LinearPartition part      = make_linear_partition(table.end[p.groups - 1], p.steps, static_cast<int>(gridDim.x), p.cutting);
    const int             worker    = static_cast<int>(blockIdx.x);

    auto locate  = [&](int tile) { return linear_locate(p, table, tile, p.nt, 16, kLinearRows, tiles_m); };
    auto columns = [&](const LinearTile& t) { return (t.rows + 15) & ~15; };

    int issued = 0;  // ring stages filled (warp 0)
    if (warp == 0) {
        // ------------------------------------------------------------ TMA
        bool     ok = true;
        int      s  = 0;
        uint32_t phase = 1;  // of the stages' "empty" barriers: the first round finds them so
        for (int i = 0; ok; i++) {
            const LinearSegment seg = linear_uniform(linear_segment(part, worker, i));
            if (seg.tile < 0)
                break;
            const LinearTile t     = linear_uniform(locate(seg.tile));
            const int        boxes = (columns(t) + p.b_box - 1) / p.b_box;
            const uint32_t   bytes = kStepBlocks * (kLinearBoxBytes + boxes * p.b_box * 128u);
#pragma unroll 1
            for (int k = seg.kb0; k < seg.kb1; k++) {
                ok = linear_wait(empty(s), phase, abort_word);
                if (!ok)
                    break;
                const uint32_t dst = smem_base + s * stage_bytes;
                if (ptx::elect_one()) {
                    ptx::mbar_arrive_expect_tx(full(s), bytes);
#pragma unroll
                    for (int h = 0; h < kStepBlocks; h++) {
                        const int x = (k * kStepBlocks + h) * 128;  // a k-block behind the end of K arrives as zeros
                        ptx::tma_load_3d(dst + h * kLinearBoxBytes, &p.a_map, x, t.m0, t.group, full(s));
                        for (int b = 0; b < boxes; b++)
                            ptx::tma_load_3d(dst + kStepBlocks * kLinearBoxBytes + h * part_bytes + b * p.b_box * 128, &p.b_map, x,
                                             t.row0 + b * p.b_box, 0, full(s));
                    }
                }
                issued++;
                if (++s == p.stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    }
    else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        bool           ok    = true;
        int            s     = 0;
        uint32_t       phase = 0, use = 0;  // use: halves of TMEM handed over
        const uint64_t a_desc0 = ptx::make_smem_desc(smem_base, 16, 1024, ptx::kSwizzle128B);
        for (int i = 0; ok; i++) {
            const LinearSegment seg = linear_uniform(linear_segment(part, worker, i));
            if (seg.tile < 0)
                break;
            const uint32_t idesc = ptx::make_idesc_f16_f32(kLinearRows, linear_uniform(columns(locate(seg.tile))), false, false)
                                   | (!EIGHT && p.bf16 ? ptx::kIdescBf16 : 0u);
            int      left   = 0;  // steps that the current half still takes
            uint32_t d_tmem = 0;
#pragma unroll 1
            for (int k = seg.kb0; k < seg.kb1; k++) {
                const bool fresh = left == 0;
                if (fresh) {
                    left   = EIGHT ? min(group_steps, seg.kb1 - k) : seg.kb1 - k;
                    d_tmem = tmem_base + (use & 1) * kGroupScales;
                    ok     = linear_wait(acc_free(use & 1), ((use >> 1) & 1) ^ 1, abort_word);
                    if (!ok)
                        break;
                }
                ok = linear_wait(full(s), phase, abort_word);
                if (!ok)
                    break;
                ptx::tc_fence_after_sync();
                const uint64_t a_desc = a_desc0 + static_cast<uint64_t>((s * stage_bytes) >> 4);
                const uint64_t b_desc = a_desc + (kStepBlocks * kLinearBoxBytes >> 4);
                left--;
                if (ptx::elect_one()) {
#pragma unroll
                    for (int h = 0; h < kStepBlocks; h++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint64_t a = a_desc + h * (kLinearBoxBytes >> 4) + j * 2, b = b_desc + h * (part_bytes >> 4) + j * 2;
                            if (EIGHT)
                                ptx::umma_f8_ss(d_tmem + h * acc_width, a, b, idesc, j > 0);
                            else
                                ptx::umma_f16_ss(d_tmem, a, b, idesc, !fresh || h > 0 || j > 0);
                        }
                    ptx::umma_commit(empty(s));
                    if (left == 0)
                        ptx::umma_commit(acc_full(use & 1));
                }
                if (EIGHT)
                    d_tmem += kStepBlocks * acc_width;
                if (left == 0)
                    use++;
                if (++s == p.stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    }
    else if (warp == 2) {
        // ------------------------------------------------------------ scales
        if (EIGHT) {
            // A group's scales are loaded two groups ahead: with the memory system busy a load takes as long as several
            // steps.  Value v of a group is k-block v / acc_width, column v % acc_width; lane l has v = l, l + 32, ...
            constexpr int PER = kGroupScales / 32;
            struct Ahead {
                float a, b[PER];
            };
            int           next_i = 0, next_k = 0;  // the segment and step that `fetch` is at
            LinearSegment next_seg = linear_segment(part, worker, 0);
            LinearTile    next_tile{};
            if (next_seg.tile >= 0) {
                next_tile = locate(next_seg.tile);
                next_k    = next_seg.kb0;
            }
            auto fetch = [&](Ahead& f) {  // false: no groups left
                if (next_seg.tile < 0)
                    return false;
                const float* sa = p.a_scales + (static_cast<size_t>(next_tile.group) * tiles_m + next_tile.m0 / kLinearRows) * p.kb;
                const int    k0 = next_k * kStepBlocks;
                // A k-block behind the end of K, the second of the last step, has the factor 0: a product of zeros times an
                // infinite scale of the block before it would be NaN.
                const int own = k0 + (lane & (kGroupBlocks - 1));
                f.a           = own < p.kb ? __ldcg(sa + own) : 0.0f;
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const int v = lane + 32 * j, block = k0 + (v >> acc_shift), column = v & (acc_width - 1);
                    f.b[j] = block < p.kb ? __ldcg(p.b_scales + static_cast<size_t>(block) * p.n + next_tile.row0 + min(column, next_tile.rows - 1))
                                          : 0.0f;
                }
                next_k += group_steps;
                if (next_k >= next_seg.kb1) {
                    next_seg = linear_segment(part, worker, ++next_i);
                    if (next_seg.tile >= 0) {
                        next_tile = locate(next_seg.tile);
                        next_k    = next_seg.kb0;
                    }
                }
                return true;
            };
            Ahead    one, two;
            uint32_t use = 0;
            auto     lay_out = [&](const Ahead& f) {
                if (!linear_wait(acc_free(use & 1), ((use >> 1) & 1) ^ 1, abort_word))
                    return false;
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const int v = lane + 32 * j;
                    scale_ring[(use & 1) * kGroupScales + v] = f.b[j] * __shfl_sync(0xffffffffu, f.a, v >> acc_shift);
                }
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(acc_full(use & 1));
                use++;
                return true;
            };
            bool have_one = fetch(one), have_two = fetch(two);
            while (have_one) {
                if (!lay_out(one))
                    break;
                have_one = fetch(one);
                if (!have_two || !lay_out(two))
                    break;
                have_two = fetch(two);
            }
        }
    }
    else if (warp >= 4) {
        // ------------------------------------------------------------ epilogue
        const int      team    = (warp - 4) >> 2;
        const int      row     = (warp & 3) * 32 + lane;  // lane of the accumulator
        const uint32_t tmem_at = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        auto           col_of  = [&](int i) { return (2 * i + team) * CH; };
        uint32_t       use     = 0;
        bool           ok      = true;
        for (int i = 0; ok; i++) {
            const LinearSegment seg = linear_segment(part, worker, i);
            if (seg.tile < 0)
                break;
            const LinearTile t = locate(seg.tile);
            const int        n = columns(t);
            float            acc[EIGHT ? NCH * CH : 1];
            if (EIGHT) {
#pragma unroll
                for (int c = 0; c < NCH * CH; c++)
                    acc[c] = 0.0f;
#pragma unroll 1
                for (int k = seg.kb0; k < seg.kb1; k += group_steps, use++) {
                    ok = linear_wait(acc_full(use & 1), (use >> 1) & 1, abort_word);
                    if (!ok)
                        break;
                    ptx::tc_fence_after_sync();
                    const int    blocks  = min(group_steps, seg.kb1 - k) * kStepBlocks;
                    uint32_t     from    = tmem_at + (use & 1) * kGroupScales;
                    const float* scales  = scale_ring + (use & 1) * kGroupScales;
#pragma unroll 1
                    for (int h = 0; h < blocks; h++, from += acc_width, scales += acc_width) {
#pragma unroll
                        for (int c = 0; c < NCH; c++) {
                            if (col_of(c) < n) {
                                uint32_t product[CH];
                                ptx::tmem_ld_x16(from + col_of(c), product);
                                ptx::tmem_ld_wait();
                                const float4* sc = reinterpret_cast<const float4*>(scales + col_of(c));
#pragma unroll
                                for (int j = 0; j < CH / 4; j++) {
                                    const float4 f = sc[j];
                                    acc[c * CH + 4 * j] += __uint_as_float(product[4 * j]) * f.x;
                                    acc[c * CH + 4 * j + 1] += __uint_as_float(product[4 * j + 1]) * f.y;
                                    acc[c * CH + 4 * j + 2] += __uint_as_float(product[4 * j + 2]) * f.z;
                                    acc[c * CH + 4 * j + 3] += __uint_as_float(product[4 * j + 3]) * f.w;
                                }
                            }
                        }
                    }
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0)
                        ptx::mbar_arrive(acc_free(use & 1));
                }
            }
            else {
                ok = linear_wait(acc_full(use & 1), (use >> 1) & 1, abort_word);
                ptx::tc_fence_after_sync();
            }
            if (!ok)
                break;
            // chunk c of this warp as fp32: out of the registers, or out of TMEM
            auto values = [&](int c, float* v) {
                if constexpr (EIGHT) {
#pragma unroll
                    for (int j = 0; j < CH; j++)
                        v[j] = acc[c * CH + j];
                }
                else {
                    uint32_t chunk[CH];
                    ptx::tmem_ld_x16(tmem_at + (use & 1) * kGroupScales + col_of(c), chunk);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < CH; j++)
                        v[j] = __uint_as_float(chunk[j]);
                }
            };
            auto store = [&](int c, const float* v) { linear_store_columns<CH>(p, t, t.m0 + row, col_of(c), v); };
            if (seg.first == seg.last) {
#pragma unroll
                for (int c = 0; c < NCH; c++)
                    if (col_of(c) < n) {
                        float v[CH];
                        values(c, v);
                        store(c, v);
                    }
            }
            else {
                // slots: [columns / 4][128 lanes] float4, so that a warp's accesses are contiguous
                const size_t  slot4 = static_cast<size_t>(kLinearRows) * p.nt / 4;
                float4* const slots = reinterpret_cast<float4*>(p.slots) + row;
                float4* const mine  = slots + worker * slot4;
#pragma unroll
                for (int c = 0; c < NCH; c++)
                    if (col_of(c) < n) {
                        float v[CH];
                        values(c, v);
#pragma unroll
                        for (int j = 0; j < CH / 4; j++)
                            __stcg(mine + (col_of(c) / 4 + j) * kLinearRows, make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
                    }
                __threadfence();
                __syncwarp();
                unsigned  arrived = 0;
                unsigned* counter = p.counters + seg.first * kEpilogueTeams + (warp - 4);
                if (lane == 0)
                    arrived = atomicAdd(counter, 1u);
                arrived = __shfl_sync(0xffffffffu, arrived, 0);
                if (arrived == static_cast<unsigned>(seg.last - seg.first)) {
                    if (lane == 0)
                        *counter = 0;  // as the next launch expects it
                    __threadfence();
#pragma unroll 1
                    for (int c = 0; c < NCH; c++)
                        if (col_of(c) < n) {
                            float v[CH];
#pragma unroll
                            for (int j = 0; j < CH; j++)
                                v[j] = 0.0f;
#pragma unroll 1
                            for (int w = seg.first; w <= seg.last; w++) {
                                const float4* from = slots + w * slot4 + (col_of(c) / 4) * kLinearRows;
#pragma unroll
                                for (int j = 0; j < CH / 4; j++) {
                                    const float4 f = __ldcg(from + j * kLinearRows);
                                    v[4 * j] += f.x;
                                    v[4 * j + 1] += f.y;
                                    v[4 * j + 2] += f.z;
                                    v[4 * j + 3] += f.w;
                                }
                            }
                            store(c, v);
                        }
                }
            }
            if (!EIGHT) {
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(acc_free(use & 1));
                use++;
            }
        }
    }

    // ---------------------------------------------------------------- exit
    ptx::tc_fence_before_sync();
    __syncthreads();
    const bool abandoned = *abort_word != 0;
    if (threadIdx.x == 0 && abandoned)
        atomicExch(&g_linear_status, 1);
    if (warp == 0 && abandoned)  // copies still under way land before the block's memory goes
        for (int i = max(0, issued - p.stages); i < issued; i++)
            ptx::mbar_wait_quiet(full(i % p.stages), (i / p.stages) & 1, kDrainNs);
    if (warp == 1) {
        if (abandoned) {  // and products end before TMEM does
            if (ptx::elect_one())
                ptx::umma_commit(drained);
            __syncwarp();
            ptx::mbar_wait_quiet(drained, 0, kDrainNs);
            __syncwarp();
        }
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace spmm_b200
