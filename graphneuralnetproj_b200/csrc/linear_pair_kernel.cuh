// The linear layers of linear_kernel.cuh at token counts where the tensor core is the bound: tiles of 256 x 256 on pairs of
// SMs (tcgen05.mma.cta_group::2, a cluster of two blocks).
//
// Per k-block (128 bytes of K) the pair MMA takes 512 cycles, in which each block has to bring in 32 KB: 128 rows of the
// operand on the accumulator's lanes and half of the 256 of the operand on its columns.  One block alone would have to
// bring in 48 KB in the same time, more than L2 hands to an SM.
//
// 16-bit operands: weights on the lanes, tokens as columns, as in the single-block kernel -- the columns of the last tile
// of a group are cut to its tokens (in steps of 32).
// Codes: tokens on the lanes, weights as columns.  Every k-block is a product of its own that the epilogue warps add to
// fp32 registers (128 of them per thread: two warpgroups share the 256 columns) while the tensor core fills the other
// half of TMEM.  This way round a thread's factor is one number per k-block, (its token's scale) * (the scale of its 128
// columns); with tokens as columns each column needs its own factor out of shared memory, which costs as much of shared
// memory's time as the operands do.
//
// What bounds them.  16 bits: the tensor core (2048 x 9472 x 4096: 111 us against 97 at the measured cuBLAS rate, tensor pipe
// active 83 %).  Codes: the way round a TMEM buffer -- MMA, commit, wake-up, read-out, additions, arrival at the leader, next MMA --
// of which there are two.  A k-block takes 0.51 us, about 840 cycles (2048 x 9472 x 8192: 149 us, tensor pipe 52 %); 0.46 without
// the TMA loads, 0.48 without the scales, 0.40 without both; the protocol by itself, on operands that stay in shared memory, takes
// 600 cycles, without the additions the 512 of the MMA.  (Additions that never stall starve the MMA warp of their scheduler: 909
// cycles; the reads out of TMEM between them prevent that.)  Measured and dropped: four warpgroups (9 % slower, bound by
// issue), 256 x 128 tiles with four buffers (8 % slower), a k-block as two products of 128 columns in four buffers (2 %
// slower), two columns per instruction (fma.rn.f32x2 runs at half rate and costs register moves), spinning instead of parked
// waits, half as many instructions around the additions (no change).
//
// Roles per block as in the single-block kernel, with warps 2 and 3 for the scales; the even block's (the leader's) warp 1
// issues the pair's MMAs, a commit arrives in both blocks.  The "full" and "acc_free" barriers live in the leader; arrivals
// there need no cluster-scope release (mbar_arrive_remote), which took over 1000 cycles each.  Every wait is bounded, and both
// blocks meet at a cluster barrier before they exit.
#pragma once

#include "linear_kernel.cuh"

namespace spmm_b200 {

constexpr int kPairTile       = 256;  // rows of A and tokens of a tile
constexpr int kPairStageBytes = 2 * kLinearBoxBytes;
constexpr int kPairStages     = 7;  // at most
constexpr int kPairBatch      = 8;  // k-blocks whose factors are handed over together

template<bool EIGHT>
__global__ void __launch_bounds__(kLinearThreads, 1)
linear_pair_kernel(const __grid_constant__ LinearParams p)
{
    constexpr int EPI = kEpilogueTeams;           // epilogue warps
    constexpr int CH  = EIGHT ? 32 : 16;          // columns per chunk
    constexpr int NCH = kPairTile / (2 * CH);     // chunks per epilogue warp

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t*       smem      = smem_raw + (smem_base - ptx::smem_addr(smem_raw));
    const uint32_t scale_off = p.stages * kPairStageBytes;  // factors: [2][kPairBatch][two halves of the columns][128 lanes]
    const uint32_t bar_off   = scale_off + (EIGHT ? 2 * kPairBatch * 1024u : 0u);
    const uint32_t bar_base  = smem_base + bar_off;
    auto full     = [&](int s) { return bar_base + 8u * s; };                        // the leader's
    auto empty    = [&](int s) { return bar_base + 8u * (kPairStages + s); };        // each block's own
    auto acc_full = [&](int b) { return bar_base + 8u * (2 * kPairStages + b); };    // each block's own
    auto acc_free = [&](int b) { return bar_base + 8u * (2 * kPairStages + 2 + b); };  // the leader's
    auto scale_full = [&](int b) { return bar_base + 8u * (2 * kPairStages + 4 + b); };  // each block's own
    auto scale_free = [&](int b) { return bar_base + 8u * (2 * kPairStages + 6 + b); };
    const uint32_t     drained = bar_base + 8u * (2 * kPairStages + 8);
    constexpr uint32_t kWords  = 8u * (2 * kPairStages + 9);
    volatile uint32_t* tmem_slot  = reinterpret_cast<volatile uint32_t*>(smem + bar_off + kWords);
    volatile int*      abort_word = reinterpret_cast<volatile int*>(smem + bar_off + kWords + 4);
    int* const         warp_sums  = reinterpret_cast<int*>(smem + bar_off + kWords + 8);
    int* const         groups_at  = reinterpret_cast<int*>(smem + bar_off + 512);
    const LinearTable  table{groups_at, groups_at + p.groups, groups_at + 2 * p.groups, groups_at + 3 * p.groups};
    static_assert(kWords + 8 + 20 * 4 <= 512, "barrier block");

    const int      warp = linear_uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_cta_rank();  // 0: leader

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; s++) {
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            ptx::mbar_init(acc_full(b), 1);
            ptx::mbar_init(acc_free(b), 2 * EPI);
            ptx::mbar_init(scale_full(b), 2);
            ptx::mbar_init(scale_free(b), EPI);
        }
        ptx::mbar_init(drained, 1);
        *abort_word = 0;
        ptx::mbar_init_fence();
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(bar_base + kWords, 512);
        ptx::tmem_relinquish_pair();
    }
    if (threadIdx.x == 0) {
        ptx::prefetch_tensor_map(&p.a_map);
        ptx::prefetch_tensor_map(&p.b_map);
    }
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const int tiles_m = (p.m - 1) / kPairTile + 1;
    ptx::tc_fence_before_sync();
    constexpr int kGranule = EIGHT ? kPairTile : 32;  // with tokens on the lanes a narrower tile costs no less
    linear_build_table<!EIGHT>(p, table, warp_sums, kPairTile, kGranule, tiles_m);
    ptx::cluster_sync_all();  // both blocks' barriers exist before anyone arrives on the partner's
    ptx::tc_fence_after_sync();
    const uint32_t        tmem_base = linear_uniform(static_cast<int>(*tmem_slot));
    const int             worker    = static_cast<int>(blockIdx.x >> 1);
    const LinearPartition part = make_linear_partition(table.end[p.groups - 1], p.steps, static_cast<int>(gridDim.x >> 1), p.cutting);

    auto locate = [&](int tile) { return linear_locate(p, table, tile, kPairTile, kGranule, kPairTile, tiles_m); };
    // columns of the accumulator that are used
    auto columns = [&](const LinearTile& t) { return EIGHT ? kPairTile : (t.rows + 31) & ~31; };

    int issued = 0;
    if (warp < 4) {
        if (EIGHT)
            ptx::registers_down<72>();
        if (warp == 0) {
            // ------------------------------------------------------------ TMA: this block's part of both operands
            bool           ok    = true;
            int            s     = 0;
            uint32_t       phase = 1;
            const uint32_t leader_full0 = ptx::map_to_cta(full(0), 0);
            for (int i = 0; ok; i++) {
                const LinearSegment seg = linear_uniform(linear_segment(part, worker, i));
                if (seg.tile < 0)
                    break;
                const LinearTile t     = linear_uniform(locate(seg.tile));
                const int        half  = columns(t) / 2;
                const int        boxes = EIGHT ? 1 : (half + p.b_box - 1) / p.b_box;
                const int        m     = t.m0 + static_cast<int>(rank) * kLinearRows;
                const int        token = t.row0 + static_cast<int>(rank) * (EIGHT ? kLinearRows : half);
                const uint32_t   bytes = 2 * (kLinearBoxBytes + (EIGHT ? kLinearBoxBytes : boxes * p.b_box * 128));
#pragma unroll 1
                for (int k = seg.kb0; k < seg.kb1; k++) {
                    ok = linear_wait(empty(s), phase, abort_word);
                    if (!ok)
                        break;
                    const uint32_t lanes = smem_base + s * kPairStageBytes, cols = lanes + kLinearBoxBytes;
                    const uint32_t bar   = leader_full0 + 8u * s;
                    if (ptx::elect_one()) {
                        if (rank == 0)
                            ptx::mbar_arrive_expect_tx(full(s), bytes);  // both blocks' bytes
                        ptx::tma_load_3d_pair(EIGHT ? cols : lanes, &p.a_map, k * 128, m, t.group, bar);
                        if (EIGHT)
                            ptx::tma_load_3d_pair(lanes, &p.b_map, k * 128, token, 0, bar);
                        else
                            for (int b = 0; b < boxes; b++)
                                ptx::tma_load_3d_pair(cols + b * p.b_box * 128, &p.b_map, k * 128, token + b * p.b_box, 0, bar);
                    }
                    issued++;
                    if (++s == p.stages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        else if (warp == 1 && rank == 0) {
            // ------------------------------------------------------------ leader: MMA for the pair
            bool           ok    = true;
            int            s     = 0;
            uint32_t       phase = 0, use = 0;
            const uint64_t desc0 = ptx::make_smem_desc(smem_base, 16, 1024, ptx::kSwizzle128B);
            for (int i = 0; ok; i++) {
                const LinearSegment seg = linear_uniform(linear_segment(part, worker, i));
                if (seg.tile < 0)
                    break;
                const uint32_t idesc = ptx::make_idesc_f16_f32(kPairTile, linear_uniform(columns(locate(seg.tile))), false, false)
                                       | (!EIGHT && p.bf16 ? ptx::kIdescBf16 : 0u);
#pragma unroll 1
                for (int k = seg.kb0; k < seg.kb1; k++) {
                    const bool fresh = EIGHT || k == seg.kb0, last = EIGHT || k == seg.kb1 - 1;
                    const bool free = !fresh || ptx::mbar_test_wait(acc_free(use & 1), ((use >> 1) & 1) ^ 1);
                    const bool here = ptx::mbar_test_wait(full(s), phase);  // asked at the same time
                    if (!__all_sync(0xffffffffu, free))
                        ok = linear_wait(acc_free(use & 1), ((use >> 1) & 1) ^ 1, abort_word);
                    if (!__all_sync(0xffffffffu, here))
                        ok = ok && linear_wait(full(s), phase, abort_word);
                    if (!ok)
                        break;
                    ptx::tc_fence_after_sync();
                    const uint32_t d_tmem = tmem_base + (use & 1) * kPairTile;
                    const uint64_t a_desc = desc0 + static_cast<uint64_t>(s * (kPairStageBytes >> 4));
                    const uint64_t b_desc = a_desc + (kLinearBoxBytes >> 4);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (EIGHT)
                                ptx::umma_f8_ss_pair(d_tmem, a_desc + j * 2, b_desc + j * 2, idesc, j > 0);
                            else
                                ptx::umma_f16_ss_pair(d_tmem, a_desc + j * 2, b_desc + j * 2, idesc, !fresh || j > 0);
                        }
                        ptx::umma_commit_both(empty(s));
                        if (last)
                            ptx::umma_commit_both(acc_full(use & 1));
                    }
                    if (last)
                        use++;
                    if (++s == p.stages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        else if (EIGHT && warp >= 2) {
            // ------------------------------------------------------------ factors: each of two warps half of a batch's k-blocks
            // (token's scale) * (scale of its 128 columns), laid out per half of the columns and lane, loaded a batch ahead.
            constexpr int PER      = kPairBatch / 2;
            const int     blocks_m = (p.m - 1) / kLinearRows + 1, mine = (warp - 2) * PER;
            float* const  ring     = reinterpret_cast<float*>(smem + scale_off);
            int           next_i = 0, next_k = 0;
            LinearSegment next_seg = linear_segment(part, worker, 0);
            LinearTile    next_tile{};
            if (next_seg.tile >= 0) {
                next_tile = locate(next_seg.tile);
                next_k    = next_seg.kb0;
            }
            float a = 0.0f, b[PER][4];  // lane 4 * h + u of `a`: columns' half h, k-block u
            auto  fetch = [&]() {
                if (next_seg.tile < 0)
                    return false;
                const int m_block = min(next_tile.m0 / kLinearRows + ((lane >> 2) & 1), blocks_m - 1);
                a = __ldcg(p.a_scales + (static_cast<size_t>(next_tile.group) * blocks_m + m_block) * p.kb
                          + min(next_k + mine + (lane & 3), p.kb - 1));
#pragma unroll
                for (int u = 0; u < PER; u++) {
                    const float* from = p.b_scales + static_cast<size_t>(min(next_k + mine + u, p.kb - 1)) * p.n + next_tile.row0;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        b[u][j] = __ldcg(from + min(static_cast<int>(rank) * kLinearRows + lane + 32 * j, next_tile.rows - 1));
                }
                next_k += kPairBatch;
                if (next_k >= next_seg.kb1) {
                    next_seg = linear_segment(part, worker, ++next_i);
                    if (next_seg.tile >= 0) {
                        next_tile = locate(next_seg.tile);
                        next_k    = next_seg.kb0;
                    }
                }
                return true;
            };
            bool have = fetch();
            for (uint32_t use = 0; have; use++) {
                if (!linear_wait(scale_free(use & 1), ((use >> 1) & 1) ^ 1, abort_word))
                    break;
#pragma unroll
                for (int u = 0; u < PER; u++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float block_scale = __shfl_sync(0xffffffffu, a, 4 * h + u);
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            ring[((use & 1) * kPairBatch + mine + u) * 256 + h * 128 + lane + 32 * j] = b[u][j] * block_scale;
                    }
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(scale_full(use & 1));
                have = fetch();
            }
        }
    }
    else {
        if (EIGHT)
            ptx::registers_up<216>();  // 128 * 72 + 256 * 216 = 384 * 168, the registers at launch
        // ------------------------------------------------------------ epilogue: this block's 128 lanes
        const int      team    = (warp - 4) >> 2;
        const int      row     = (warp & 3) * 32 + lane;
        const uint32_t tmem_at = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t leader_acc_free0 = ptx::map_to_cta(acc_free(0), 0);
        auto           col_of  = [&](int c) { return EIGHT ? (team * NCH + c) * CH : (2 * c + team) * CH; };
        uint32_t       use     = 0, batch = 0;
        bool           ok      = true;
        for (int i = 0; ok; i++) {
            const LinearSegment seg = linear_segment(part, worker, i);
            if (seg.tile < 0)
                break;
            const LinearTile t = locate(seg.tile);
            const int        n = columns(t);
            const int        token = static_cast<int>(rank) * kLinearRows + row;  // of this lane (codes)
            float            acc[EIGHT ? NCH * CH : 1];
            if constexpr (EIGHT) {
#pragma unroll
                for (int c = 0; c < NCH * CH; c++)
                    acc[c] = 0.0f;
                const float* const factors = reinterpret_cast<const float*>(smem + scale_off) + team * 128 + row;
                auto               release = [&]() {  // a batch of factors
                    __syncwarp();
                    if (lane == 0)
                        ptx::mbar_arrive(scale_free(batch & 1));
                    batch++;
                };
                auto factor_of = [&](int at) {  // of the segment's k-block `at`; asked for in order
                    if (at % kPairBatch == 0) {
                        if (at > 0)
                            release();
                        ok = linear_wait(scale_full(batch & 1), (batch >> 1) & 1, abort_word);
                    }
                    return factors[((batch & 1) * kPairBatch + at % kPairBatch) * 256];
                };
                float factor = factor_of(0);
                bool  here   = false;  // the product is known to be there
#pragma unroll 1
                for (int k = seg.kb0; k < seg.kb1 && ok; k++, use++) {
                    if (!__all_sync(0xffffffffu, here)) {
                        ok = linear_wait(acc_full(use & 1), (use >> 1) & 1, abort_word);
                        if (!ok)
                            break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t from = tmem_at + (use & 1) * kPairTile;
                    const float    f    = factor;
#pragma unroll
                    for (int c = 0; c < NCH; c++) {
                        uint32_t product[CH];
                        ptx::tmem_ld_x32_now(from + col_of(c), product);
                        if (c == NCH - 1) {
                            ptx::tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0)
                                ptx::mbar_arrive_remote(leader_acc_free0 + 8u * (use & 1));
                            // what the next k-block needs is asked for before these additions
                            here = ptx::mbar_test_wait(acc_full((use + 1) & 1), ((use + 1) >> 1) & 1);
                            if (k + 1 < seg.kb1)
                                factor = factor_of(k + 1 - seg.kb0);
                        }
#pragma unroll
                        for (int j = 0; j < CH; j++)
                            acc[c * CH + j] += __uint_as_float(product[j]) * f;
                    }
                }
                release();
            }
            else {
                ok = linear_wait(acc_full(use & 1), (use >> 1) & 1, abort_word);
                ptx::tc_fence_after_sync();
            }
            if (!ok)
                break;
            auto values = [&](int c, float* v) {
                if constexpr (EIGHT) {
#pragma unroll
                    for (int j = 0; j < CH; j++)
                        v[j] = acc[c * CH + j];
                }
                else {
                    uint32_t chunk[CH];
                    ptx::tmem_ld_x16(tmem_at + (use & 1) * kPairTile + col_of(c), chunk);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < CH; j++)
                        v[j] = __uint_as_float(chunk[j]);
                }
            };
            auto store = [&](int c, const float* v) {
                if constexpr (EIGHT) {  // one token's columns
                    const int m = t.m0 + col_of(c);
                    if (m >= p.m)
                        return;
                    if (p.wide_c) {
                        // Four neighbouring lanes exchange 16-byte pieces, so that each store of theirs is 64 contiguous bytes of one
                        // token: with 16 bytes of 32 tokens in every store the end of a tile took 3.3 us, six k-blocks' time.
                        static_assert(CH == 32, "four pieces per lane");
                        uint32_t q[4][4];
#pragma unroll
                        for (int j = 0; j < CH / 2; j++)
                            q[j / 4][j % 4] = linear_pair_of(v[2 * j], v[2 * j + 1], p.bf16);
#pragma unroll
                        for (int d = 1; d < 4; d <<= 1)
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                if (!(j & d))
#pragma unroll
                                    for (int w = 0; w < 4; w++) {
                                        const uint32_t got = __shfl_xor_sync(0xffffffffu, (lane & d) ? q[j][w] : q[j | d][w], d);
                                        q[j][w]     = (lane & d) ? got : q[j][w];
                                        q[j | d][w] = (lane & d) ? q[j | d][w] : got;
                                    }
                        const int piece = m + 8 * (lane & 3), first = token - (lane & 3);
                        uint16_t* to = static_cast<uint16_t*>(p.C) + static_cast<size_t>(t.row0 + first) * p.m + piece;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (first + j < t.rows && piece < p.m)
                                *reinterpret_cast<uint4*>(to + static_cast<size_t>(j) * p.m) = make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]);
                        return;
                    }
                    if (token < t.rows) {
                        const size_t at = static_cast<size_t>(t.row0 + token) * p.m + m;
#pragma unroll
                        for (int j = 0; j < CH; j++)
                            if (m + j < p.m)
                                linear_store(p, at + j, v[j]);
                    }
                    return;
                }
                linear_store_columns<CH>(p, t, t.m0 + static_cast<int>(rank) * kLinearRows + row, col_of(c), v);
            };
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
                constexpr size_t kSlot4 = static_cast<size_t>(kLinearRows) * kPairTile / 4;
                float4* const    slots  = reinterpret_cast<float4*>(p.slots) + rank * kSlot4 + row;
                float4* const    mine   = slots + static_cast<size_t>(2 * worker) * kSlot4;
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
                unsigned* counter = p.counters + (2 * seg.first + rank) * EPI + (warp - 4);
                if (lane == 0)
                    arrived = atomicAdd(counter, 1u);
                arrived = __shfl_sync(0xffffffffu, arrived, 0);
                if (arrived == static_cast<unsigned>(seg.last - seg.first)) {
                    if (lane == 0)
                        *counter = 0;
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
                                const float4* from = slots + static_cast<size_t>(2 * w) * kSlot4 + (col_of(c) / 4) * kLinearRows;
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
                    ptx::mbar_arrive_remote(leader_acc_free0 + 8u * (use & 1));
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
    if (abandoned && rank == 0 && warp == 0)  // both blocks' copies still under way are counted here
        for (int i = max(0, issued - p.stages); i < issued; i++)
            ptx::mbar_wait_quiet(full(i % p.stages), (i / p.stages) & 1, kDrainNs);
    if (abandoned && rank == 0 && warp == 1) {  // and products end before TMEM does
        if (ptx::elect_one())
            ptx::umma_commit_pair(ptx::map_to_cta(drained, 0));
        __syncwarp();
        ptx::mbar_wait_quiet(drained, 0, kDrainNs);
        __syncwarp();
    }
    if (abandoned && rank == 1 && warp == 0)  // copies that the leader no longer counts: it has given up on them
        ptx::mbar_wait_quiet(drained, 0, kDrainNs);  // of this block: nothing arrives on it
    // Neither block leaves while its partner may still arrive on its barriers or the leader's MMAs read its memory.
    ptx::cluster_sync_all();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

}  // namespace spmm_b200
