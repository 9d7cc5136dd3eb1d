// Dispatcher of the linear layers on dense weights (linear_kernel.cuh): 8-bit block-scaled weights, one matrix per group
// of tokens (experts), or both.  Declared in include/spmm_b200.h.
#include <algorithm>
#include <mutex>

#include "../../include/spmm_b200.h"
#include "linear_api.h"
#include "linear_kernel.cuh"

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
    int    kb;
    int    nt, b_box;
    size_t slot_bytes;
};

bool aligned16(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// Tokens per tile.  One matrix: as few tiles as 128 columns allow, of equal width.  Groups, whose sizes the host does
// not know: twice the average, so that most groups are one tile and its ring stages are not mostly unused.
void choose_tiles(LinearShape& s)
{
    s.kb = (s.k * (s.eight ? 1 : 2) - 1) / 128 + 1;
    if (!s.ragged) {
        const int tiles = std::max(1, (s.n - 1) / 128 + 1);
        s.nt            = std::max(16, ((s.n - 1) / tiles + 1 + 15) / 16 * 16);
        s.b_box         = s.nt;
    }
    else {
        const long want = std::min<long>(s.n, 2L * s.n / s.groups);
        s.nt            = want <= 16 ? 16 : (want <= 32 ? 32 : (want <= 64 ? 64 : 128));
        s.b_box         = std::min(s.nt, 32);
    }
    s.slot_bytes = static_cast<size_t>(kLinearRows) * s.nt * sizeof(float);
}

size_t workspace_needed(const LinearShape& s)
{
    return kCounterBytes + 2 * static_cast<size_t>(kMaxWorkers) * s.slot_bytes;
}

// Sizes that the format and the index arithmetic can describe.
bool valid_shape(const LinearShape& s)
{
    if (s.m < 1 || s.n < 0 || s.k < 1 || s.groups < 1 || s.groups > kLinearMaxGroups || s.k > (1 << 29) || s.k % (s.eight ? 16 : 8) != 0)
        return false;
    return true;
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

struct LinearDevice {
    int  sm_count     = 0;
    bool attrs_set[2] = {};
};

template<bool EIGHT>
cudaError_t launch(cudaStream_t stream, LinearParams& p, const LinearShape& s)
{
    int         device = 0;
    cudaError_t e      = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    static LinearDevice devices[64];
    static std::mutex   lock;
    auto                kern = linear_kernel<EIGHT>;
    int                 sms  = 0;
    {
        std::lock_guard<std::mutex> guard(lock);
        LinearDevice& d = devices[device & 63];
        if (d.sm_count == 0) {
            e = cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, device);
            if (e != cudaSuccess)
                return e;
        }
        if (!d.attrs_set[EIGHT]) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamicSmem);
            if (e != cudaSuccess) {
                (void)cudaGetLastError();
                return e;
            }
            d.attrs_set[EIGHT] = true;
        }
        sms = d.sm_count;
    }
    const int stage_bytes = kStepBlocks * (kLinearBoxBytes + s.nt * 128);
    const int fixed       = kLinearFixedSmem + (EIGHT ? 2 * kGroupScales * 4 : 0) + s.groups * 12;
    p.stages              = std::min(kLinearMaxStages, (kMaxDynamicSmem - fixed) / stage_bytes);

    cudaLaunchConfig_t config = {};
    config.gridDim            = dim3(std::min(sms, kMaxWorkers));
    config.blockDim           = dim3(kLinearThreads);
    config.dynamicSmemBytes   = fixed + p.stages * stage_bytes;
    config.stream             = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs                                       = attr;
    config.numAttrs                                    = 1;
    e = cudaLaunchKernelEx(&config, kern, p);
    return e != cudaSuccess ? e : cudaGetLastError();
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
    const long tiles_m = (s.m - 1) / kLinearRows + 1, tiles_n = (s.n - 1) / s.nt + 1;
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
    p.steps    = (s.kb - 1) / kStepBlocks + 1;
    p.nt       = s.nt;
    p.b_box    = s.b_box;
    p.bf16     = C_type == SPMM_B200_BF16;
    p.overhead = -1;
    if (workspace && workspace_bytes >= workspace_needed(s)) {
        p.counters = static_cast<unsigned*>(workspace);
        p.slots    = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
        p.overhead = 2;
    }
    return s.eight ? launch<true>(stream, p, s) : launch<false>(stream, p, s);
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

int linear_status(int reset)
{
    int         status = 0;
    cudaError_t e      = cudaMemcpyFromSymbol(&status, g_linear_status, sizeof(int));
    if (e != cudaSuccess)
        return -static_cast<int>(e);
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

int spmm_b200_linear_plan(int tiles, int kb, int workers, int overhead, int worker, int index, int* segment)
{
    using namespace spmm_b200;
    if (tiles < 0 || kb < 1 || workers < 1 || worker < 0 || worker >= workers || index < 0 || !segment)
        return static_cast<int>(cudaErrorInvalidValue);
    const LinearPartition p = make_linear_partition(tiles, kb, workers, overhead);
    const LinearSegment   s = linear_segment(p, worker, index);
    segment[0] = s.tile;
    segment[1] = s.kb0;
    segment[2] = s.kb1;
    segment[3] = s.slot;
    segment[4] = s.first;
    segment[5] = s.last;
    segment[6] = s.tile >= 0 && s.slot >= 0 ? linear_slot_of(p, s, worker) : -1;
    return static_cast<int>(cudaSuccess);
}

}  // extern "C"
