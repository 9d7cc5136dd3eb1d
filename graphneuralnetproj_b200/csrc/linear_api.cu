// Dispatcher of the linear layers on dense weights (linear_kernel.cuh): 8-bit block-scaled weights, one matrix per group
// of tokens (experts), or both.  Declared in include/spmm_b200.h.
#include <algorithm>
#include <mutex>

#include "../../include/spmm_b200.h"
#include "linear_api.h"
#include "linear_kernel.cuh"
#include "linear_pair_kernel.cuh"

namespace spmm_b200 {
namespace {

constexpr int    kMaxWorkers     = 148;  // blocks of a launch: one per SM
constexpr size_t kCounterBytes   = kPieceCounters * sizeof(unsigned);
constexpr int    kMaxDynamicSmem = 227 * 1024;

struct LinearShape {
    bool eight;
    int  groups, m, n, k;
    bool ragged;  // group borders are read on the device

    // What follows from the sizes:
    bool   pair;        // tiles of 256 x 256 on pairs of SMs
    int    kb;          // k-blocks
    int    nt, b_box;   // tokens per tile, and per TMA box
    size_t slot_bytes;  // a worker's piece of a tile
};

bool aligned16(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// Which kernel, and tokens per tile.  One block per tile takes 128 tokens at most.  All tokens of one matrix fit a tile then
// (there would be pairs with more of them); the tokens of groups, whose sizes the host does not know, are cut into tiles of
// twice the average, so that most groups are one tile and its ring stages are not mostly unused.
void choose_tiles(LinearShape& s)
{
    s.kb            = (s.k * (s.eight ? 1 : 2) - 1) / 128 + 1;
    const int group = s.ragged ? s.n / s.groups : s.n;  // tokens, on average
    s.pair          = group > 128;
    if (s.pair) {
        s.nt         = kPairTile;
        s.b_box      = s.eight ? kLinearRows : 64;
        s.slot_bytes = 2 * static_cast<size_t>(kLinearRows) * kPairTile * sizeof(float);
        return;
    }
    if (!s.ragged) {
        s.nt    = (s.n + 15) / 16 * 16;
        s.b_box = s.nt;
    }
    else {
        const long want = std::min<long>(s.n, 2L * s.n / s.groups);
        s.nt            = want <= 16 ? 16 : (want <= 32 ? 32 : (want <= 64 ? 64 : 128));
        s.b_box         = std::min(s.nt, 32);
    }
    s.slot_bytes = static_cast<size_t>(kLinearRows) * s.nt * sizeof(float);
}

int max_workers(const LinearShape& s)
{
    return s.pair ? kMaxWorkers / 2 : kMaxWorkers;
}

// What cutting a tile costs (linear_plan.h), in steps (k-blocks of pairs), from measurements of whole and cut tiles.  It depends
// on the width: a step of 16 bits has half the features, and no additions on its way.  Times in us, weights m x k.
//   up to 32 tokens     8 bits  16 x 2048 x 4096 (16 steps): 11.4 whole, 10.2 cut;  16 x 4096 x 2048 (8): 8.2 and 9.3
//                      16 bits  16 x 4096 x 4096 (32): 16.2 and 12.3;  16 x 4096 x 2048 (16): 10.0 and 9.5
//   up to 64            8 bits  33 x 7168 x 7168 (28): 20.0 and 18.2;  64 x 2048 x 4096 (16): 13.4 and 12.3;  64 x 4096 x 2048 (8): 9.5 and 11.2
//                      16 bits  64 x 7168 x 7168 (56): 28.4 and 25.9;  61 x 320 x 2880 (23): 13.8 and 11.1;  33 x 4096 x 2048 (16): 11.2 and 11.6
//   up to 128           8 bits  100 x 7168 x 7168 (28): 29.8 and 23.7;  128 x 4096 x 4096 (16): 20.0 and 18.4;  128 x 4096 x 2048 (8): 12.5 and 14.6
//                      16 bits  100 x 7168 x 7168 (56): 32.3 and 29.8;  137 over 2 x 2640 x 4304 (34): 23.9 and 21.4;  128 x 4096 x 2048 (16): 12.0 and 15.2
//   pairs               8 bits  200 x 7168 x 7168 (56): 32.5 and 28.4;  512 x 4096 x 4096 (32): 21.4 and 22.5
//                      16 bits  200 x 1024 x 8192 (128): 38.2 and 30.5;  200 x 7168 x 7168 (112): 36.2 and 37.5;  200 x 4096 x 2048 (32): 15.5 and 27.3
LinearCutting cutting(const LinearShape& s)
{
    if (s.pair)
        return LinearCutting{s.eight ? 18 : 62, 4};
    if (s.nt <= 32)
        return LinearCutting{9, 16};
    if (s.nt <= 64)
        return LinearCutting{s.eight ? 9 : 12, 16};
    return LinearCutting{s.eight ? 8 : 20, 16};
}

size_t workspace_needed(const LinearShape& s)
{
    return kCounterBytes + static_cast<size_t>(max_workers(s)) * s.slot_bytes;
}

// Sizes that the format and the index arithmetic can describe.  Tokens: the columns of the last tile behind the last token
// have numbers too, which have to fit an int.  Depth: the byte offset in a row has to; with 16 bits the whole depth of a tile is
// one accumulation (half a microsecond per 64) that the epilogue waits for, and a wait gives up after two seconds.
constexpr int kMaxTokens  = 0x7fffffff - 2 * kPairTile;
constexpr int kMaxDepth8  = 1 << 29;
constexpr int kMaxDepth16 = 1 << 27;

bool valid_shape(const LinearShape& s)
{
    return s.m >= 1 && s.n >= 0 && s.n <= kMaxTokens && s.k >= 1 && s.k <= (s.eight ? kMaxDepth8 : kMaxDepth16) && s.k % (s.eight ? 16 : 8) == 0
           && s.groups >= 1 && s.groups <= kLinearMaxGroups;
}

cudaError_t describe(CUtensorMap& map, const void* base, long row_bytes, long rows, long groups, int box_rows)
{
    using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn   encode = nullptr;
    static std::mutex lock;
    {
        std::lock_guard<std::mutex> guard(lock);
        if (encode == nullptr) {
            void*                           fn     = nullptr;
            cudaDriverEntryPointQueryResult status = cudaDriverEntryPointSymbolNotFound;
            cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &status);
            if (e != cudaSuccess || status != cudaDriverEntryPointSuccess || fn == nullptr)
                return e != cudaSuccess ? e : cudaErrorNotSupported;
            encode = reinterpret_cast<EncodeFn>(fn);
        }
    }
    const cuuint64_t dims[3]    = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(groups)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(row_bytes) * rows};
    const cuuint32_t box[3]     = {128, static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t steps[3]   = {1, 1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                   == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

// What is looked up once per device and kernel: the blocks (or pairs) that run at the same time.
struct LinearDevice {
    int workers[4] = {};
};

template<bool EIGHT, bool PAIR>
cudaError_t launch(cudaStream_t stream, LinearParams& p, const LinearShape& s)
{
    int         device = 0;
    cudaError_t e      = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    auto      kern        = PAIR ? linear_pair_kernel<EIGHT> : linear_kernel<EIGHT>;
    const int stage_bytes = PAIR ? kPairStageBytes : kStepBlocks * (kLinearBoxBytes + s.nt * 128);
    const int fixed       = kLinearFixedSmem + (EIGHT ? (PAIR ? 2 * kPairBatch * 1024 : 2 * kGroupScales * 4) : 0) + s.groups * kLinearTableWords * 4;
    p.stages              = std::min(PAIR ? kPairStages : kLinearMaxStages, (kMaxDynamicSmem - fixed) / stage_bytes);
    p.steps               = PAIR ? s.kb : (s.kb - 1) / kStepBlocks + 1;

    cudaLaunchConfig_t config = {};
    config.blockDim           = dim3(kLinearThreads);
    config.dynamicSmemBytes   = fixed + p.stages * stage_bytes;
    config.stream             = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id                                         = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x                           = 2;
    attr[1].val.clusterDim.y                           = 1;
    attr[1].val.clusterDim.z                           = 1;
    config.attrs                                       = attr;
    config.numAttrs                                    = PAIR ? 2 : 1;

    static LinearDevice devices[64];
    static std::mutex   lock;
    int                 workers = 0;
    {
        std::lock_guard<std::mutex> guard(lock);
        int& known = devices[device & 63].workers[2 * PAIR + EIGHT];
        if (known == 0) {
            int sms = 0, found = 0;
            e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamicSmem);
            if (e == cudaSuccess && PAIR) {
                cudaLaunchConfig_t probe = config;
                probe.gridDim            = dim3(sms / 2 * 2);
                probe.dynamicSmemBytes   = kMaxDynamicSmem;
                probe.attrs              = attr + 1;
                probe.numAttrs           = 1;
                e                        = cudaOccupancyMaxActiveClusters(&found, kern, &probe);
            }
            if (e != cudaSuccess) {
                (void)cudaGetLastError();  // do not leave the error behind for an unrelated later call
                return e;
            }
            found = std::min(PAIR ? std::min(found, sms / 2) : sms, max_workers(s));
            if (found < 1)
                return cudaErrorNotSupported;
            known = found;
        }
        workers = known;
    }
    config.gridDim = dim3(PAIR ? 2 * workers : workers);
    e              = cudaLaunchKernelEx(&config, kern, p);
    if (e != cudaSuccess)
        (void)cudaGetLastError();
    return e;  // not what an earlier call has left behind
}

cudaError_t linear(cudaStream_t stream, LinearShape s, const void* A, const float* A_scales, const void* B, const float* B_scales, void* C,
                   int C_type, const int* offsets, void* workspace, size_t workspace_bytes)
{
    if (!valid_shape(s) || (C_type != SPMM_B200_FP16 && C_type != SPMM_B200_BF16))
        return cudaErrorInvalidValue;
    if (s.n == 0)
        return cudaSuccess;
    if (!A || !B || !C || (s.eight && (!A_scales || !B_scales)) || (s.ragged && !offsets) || !aligned16(A) || !aligned16(B)
        || (reinterpret_cast<uintptr_t>(C) & 1u) || !aligned16(workspace)
        || ((reinterpret_cast<uintptr_t>(A_scales) | reinterpret_cast<uintptr_t>(B_scales) | reinterpret_cast<uintptr_t>(offsets)) & 3u))
        return cudaErrorInvalidValue;
    choose_tiles(s);
    // even a table of borders that is corrupt must not overflow the tile numbers
    const long tiles_m = (s.m - 1) / (s.pair ? kPairTile : kLinearRows) + 1, tiles_n = (s.n - 1) / s.nt + 1;
    if (tiles_m * tiles_n > 0x7fffffffL / s.groups)
        return cudaErrorInvalidValue;

    LinearParams p = {};
    const long   row_bytes = static_cast<long>(s.k) * (s.eight ? 1 : 2);
    cudaError_t  e         = describe(p.a_map, A, row_bytes, s.m, s.groups, kLinearRows);
    if (e == cudaSuccess)
        e = describe(p.b_map, B, row_bytes, s.n, 1, s.b_box);
    if (e != cudaSuccess)
        return e;
    p.a_scales = A_scales;
    p.b_scales = B_scales;
    p.C        = C;
    p.offsets  = s.ragged ? offsets : nullptr;
    p.groups   = s.groups;
    p.m        = s.m;
    p.n        = s.n;
    p.kb       = s.kb;
    p.nt       = s.nt;
    p.b_box    = s.b_box;
    p.bf16     = C_type == SPMM_B200_BF16;
    p.cutting  = cutting(s);
    if (workspace && workspace_bytes >= workspace_needed(s)) {
        p.counters = static_cast<unsigned*>(workspace);
        p.slots    = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    }
    else
        p.cutting.overhead = -1;
    p.wide_c = aligned16(C) && s.m % 8 == 0;
    if (s.pair)
        return s.eight ? launch<true, true>(stream, p, s) : launch<false, true>(stream, p, s);
    return s.eight ? launch<true, false>(stream, p, s) : launch<false, false>(stream, p, s);
}

LinearShape shape_of(bool eight, bool ragged, int groups, int m, int n, int k)
{
    LinearShape s = {};
    s.eight       = eight;
    s.ragged      = ragged;
    s.groups      = groups;
    s.m           = m;
    s.n           = n;
    s.k           = k;
    return s;
}

}  // namespace

// Two warps wait for a phase of a barrier that nothing completes: the first to reach the limit gives up, the other follows its
// abort word, each as a whole (the vote after the wait takes part of all lanes), and the block ends normally.
__global__ void linear_wait_that_runs_out_kernel(uint64_t limit_ns)
{
    __shared__ __align__(8) uint64_t bar;
    __shared__ int                   abort_word;
    if (threadIdx.x == 0) {
        ptx::mbar_init(ptx::smem_addr(&bar), 1);
        ptx::mbar_init_fence();
        abort_word = 0;
    }
    __syncthreads();
    // warp 1 alone could wait as long as any wait of the kernels
    const bool ok = linear_wait(ptx::smem_addr(&bar), 0, &abort_word, threadIdx.x < 32 ? limit_ns : ptx::kWaitLimitNs);
    const bool all_gave_up = __all_sync(0xffffffffu, !ok);
    __syncthreads();
    if (threadIdx.x == 32 && all_gave_up && abort_word != 0)
        atomicExch(&g_linear_status, 1);
}

int linear_status(int reset)
{
    int         status = 0;
    cudaError_t e      = cudaMemcpyFromSymbol(&status, g_linear_status, sizeof(int));
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return -static_cast<int>(e);
    }
    if (reset) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int));
    }
    return status;
}

}  // namespace spmm_b200

// ------------------------------------------------------------------ extern "C"
extern "C" {

size_t spmm_b200_linear_workspace_bytes(int groups, int M_Global, int N_Global, int K_Global, int eight_bit)
{
    using namespace spmm_b200;
    // a call with one group and a call without group borders may take different tiles: the larger of the two
    size_t most = 0;
    for (int ragged = groups == 1 ? 0 : 1; ragged < 2; ragged++) {
        LinearShape s = shape_of(eight_bit != 0, ragged != 0, groups, M_Global, N_Global, K_Global);
        if (!valid_shape(s))
            return 0;
        if (s.n > 0) {
            choose_tiles(s);
            most = std::max(most, workspace_needed(s));
        }
    }
    return most;
}

int spmm_b200_fp8_linear(void*        stream,
                         const void*  A,
                         const float* A_scales,
                         const void*  B,
                         const float* B_scales,
                         void*        C,
                         int          C_type,
                         int          M_Global,
                         int          N_Global,
                         int          K_Global,
                         void*        workspace,
                         size_t       workspace_bytes)
{
    using namespace spmm_b200;
    return static_cast<int>(linear(static_cast<cudaStream_t>(stream), shape_of(true, false, 1, M_Global, N_Global, K_Global), A, A_scales, B,
                                   B_scales, C, C_type, nullptr, workspace, workspace_bytes));
}

int spmm_b200_grouped_linear(void*       stream,
                             const void* A,
                             const void* B,
                             void*       C,
                             int         type,
                             const int*  group_offsets,
                             int         groups,
                             int         M_Global,
                             int         N_Global,
                             int         K_Global,
                             void*       workspace,
                             size_t      workspace_bytes)
{
    using namespace spmm_b200;
    return static_cast<int>(linear(static_cast<cudaStream_t>(stream), shape_of(false, true, groups, M_Global, N_Global, K_Global), A, nullptr, B,
                                   nullptr, C, type, group_offsets, workspace, workspace_bytes));
}

int spmm_b200_grouped_fp8_linear(void*        stream,
                                 const void*  A,
                                 const float* A_scales,
                                 const void*  B,
                                 const float* B_scales,
                                 void*        C,
                                 int          C_type,
                                 const int*   group_offsets,
                                 int          groups,
                                 int          M_Global,
                                 int          N_Global,
                                 int          K_Global,
                                 void*        workspace,
                                 size_t       workspace_bytes)
{
    using namespace spmm_b200;
    return static_cast<int>(linear(static_cast<cudaStream_t>(stream), shape_of(true, true, groups, M_Global, N_Global, K_Global), A, A_scales,
                                   B, B_scales, C, C_type, group_offsets, workspace, workspace_bytes));
}

int spmm_b200_selftest_linear_wait_timeout(void* stream, unsigned int limit_ms)
{
    if (limit_ms == 0 || limit_ms > 1000)
        return static_cast<int>(cudaErrorInvalidValue);
    cudaLaunchConfig_t config = {};
    config.gridDim            = dim3(1);
    config.blockDim           = dim3(64);
    config.stream             = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaLaunchKernelEx(&config, spmm_b200::linear_wait_that_runs_out_kernel, static_cast<uint64_t>(limit_ms) * 1000000ull);
    if (e != cudaSuccess)
        (void)cudaGetLastError();
    return static_cast<int>(e);
}

int spmm_b200_linear_plan(int tiles, int kb, int workers, int overhead, int pieces, int worker, int index, int* segment)
{
    using namespace spmm_b200;
    if (tiles < 0 || kb < 1 || workers < 1 || pieces < 1 || worker < 0 || worker >= workers || index < 0 || !segment)
        return static_cast<int>(cudaErrorInvalidValue);
    const LinearPartition p = make_linear_partition(tiles, kb, workers, LinearCutting{overhead, pieces});
    const LinearSegment   s = linear_segment(p, worker, index);
    segment[0] = s.tile;
    segment[1] = s.kb0;
    segment[2] = s.kb1;
    segment[3] = s.first;
    segment[4] = s.last;
    return static_cast<int>(cudaSuccess);
}

}  // extern "C"
