// Block-scaled 8-bit values (e4m3) from fp16 or bf16 ones: the operands of the 8-bit linear layers (linear_api.cu).
//
//   s = max(amax / 448, 2^-64)   one fp32 scale per block, amax over the block's finite elements
//   c = e4m3(x / s)              the e4m3 value nearest to the exact quotient, ties to even
//
// Blocks are 1 x 128 along a row (activations: one scale per token and 128 features) or 128 x 128 (weights).  448 is
// the largest e4m3 value, so amax maps to it; the floor keeps the scale of an all-zero block usable and every
// quotient clear of fp32's subnormals.  e4m3 has no infinity: an element that is infinite or NaN becomes NaN, which
// reaches every result that uses it, and its neighbours in the block are scaled as if it were not there.
//
// Rounding to the nearest value of the *exact* quotient: x is multiplied by a number a little below 1 / s and by one a
// little above, so that the exact quotient lies between the two products.  Rounding never changes the order of two numbers:
// where both products get the same code, the quotient has it too.  Otherwise the quotient is next to the midpoint m of the
// two codes' values, and x - m * s, whose sign one fused multiply-add gives exactly, says on which side.  That is no rare
// case: two bf16 numbers of eight bits often have a ratio that is a midpoint but for the rounding of s (one element in 200;
// fp16: one in 1500), so it has to be cheap as well: with none of them 4099 x 12288 would take 26 us.
//
// Bound by memory (2 bytes in, 1 out per element) only if an element costs less than about ten instructions.  Dividing, or
// looking at the product's bits for the neighbourhood of a midpoint (and differently below the smallest normal e4m3 value),
// costs two to three times that; 16 elements per lane halve the shuffles and index arithmetic of 8.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/spmm_b200.h"
#include "ptx_sm100.cuh"

namespace spmm_b200 {
namespace {

constexpr float kE4m3Max  = 448.0f;
constexpr float kScaleMin = 5.42101086242752217e-20f;  // 2^-64
constexpr int   kBlock    = 128;

template<bool BF16>
__device__ __forceinline__ float element(uint32_t bits16)
{
    if (BF16)
        return __uint_as_float(bits16 << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
}

// The pattern of the smallest magnitude that is not finite, in both halves.
template<bool BF16>
constexpr uint32_t kInfPair = BF16 ? 0x7f807f80u : 0x7c007c00u;

// Largest magnitude of the elements seen, as the 16-bit pattern of its absolute value (patterns of the same sign order like
// the numbers; infinities and NaN come last), per half.
__device__ __forceinline__ uint32_t amax_bits(uint32_t m, uint4 v)
{
    m = __vmaxu2(m, v.x & 0x7fff7fffu);
    m = __vmaxu2(m, v.y & 0x7fff7fffu);
    m = __vmaxu2(m, v.z & 0x7fff7fffu);
    return __vmaxu2(m, v.w & 0x7fff7fffu);
}

// Elements that are not finite, as zeros.
template<bool BF16>
__device__ __forceinline__ uint32_t finite_only(uint32_t v)
{
    return v & ~__vcmpgeu2(v & 0x7fff7fffu, kInfPair<BF16>);
}
template<bool BF16>
__device__ __forceinline__ uint4 finite_only(uint4 v)
{
    return make_uint4(finite_only<BF16>(v.x), finite_only<BF16>(v.y), finite_only<BF16>(v.z), finite_only<BF16>(v.w));
}

template<bool BF16>
__device__ __forceinline__ float scale_of(uint32_t amax16)
{
    return fmaxf(__fdiv_rn(element<BF16>(amax16), kE4m3Max), kScaleMin);
}

// Four codes, the first in the lowest byte.
__device__ __forceinline__ uint32_t e4m3_quad(float x0, float x1, float x2, float x3)
{
    uint32_t out;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(out)
        : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
    return out;
}

// A block's scale, and the factors a little below and above 1 / scale.
struct BlockScale {
    float scale, below, above;
};

__device__ __forceinline__ BlockScale block_scale(float scale)
{
    // 1 / scale is off by half a unit in the last place, a product with it by another half: two units more or less bound both
    const int inv = __float_as_int(__frcp_rn(scale));
    return BlockScale{scale, __int_as_float(inv - 2), __int_as_float(inv + 2)};
}

// The codes of four quotients x / s that lie between the values of `lo` and `hi` (neighbours, or the same), all four bytes at
// once: on magnitudes, the quotient has the farther code if x - m * s is positive, or zero and that code is even.
__device__ __forceinline__ uint32_t settle(uint32_t lo, uint32_t hi, const float* x, float s)
{
    uint32_t take = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t a, b;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(static_cast<uint16_t>((lo & 0x7f7f7f7fu) >> (16 * i))));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(static_cast<uint16_t>((hi & 0x7f7f7f7fu) >> (16 * i))));
        const float2 sum = __half22float2(__hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b)));
        const int    r0  = __float_as_int(__fmaf_rn(sum.x, -0.5f * s, fabsf(x[2 * i])));
        const int    r1  = __float_as_int(__fmaf_rn(sum.y, -0.5f * s, fabsf(x[2 * i + 1])));
        take |= r0 >= static_cast<int>((hi >> (16 * i)) & 1u) ? 0xffu << (16 * i) : 0u;
        take |= r1 >= static_cast<int>((hi >> (16 * i + 8)) & 1u) ? 0xff00u << (16 * i) : 0u;
    }
    return (hi & take) | (lo & ~take);
}

// Eight elements to eight codes.  redo: the block holds elements that are not finite (all their bits set they are NaN).
template<bool BF16>
__device__ __forceinline__ uint2 encode8(uint4 v, BlockScale s, bool redo)
{
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (redo) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] |= __vcmpgeu2(w[i] & 0x7fff7fffu, kInfPair<BF16>);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i]     = element<BF16>(w[i] & 0xffffu);
        x[2 * i + 1] = element<BF16>(w[i] >> 16);
    }
    uint32_t lo[2], hi[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float* y = x + 4 * i;
        lo[i] = e4m3_quad(y[0] * s.below, y[1] * s.below, y[2] * s.below, y[3] * s.below);
        hi[i] = e4m3_quad(y[0] * s.above, y[1] * s.above, y[2] * s.above, y[3] * s.above);
    }
    if (lo[0] != hi[0])
        lo[0] = settle(lo[0], hi[0], x, s.scale);
    if (lo[1] != hi[1])
        lo[1] = settle(lo[1], hi[1], x + 4, s.scale);
    return make_uint2(lo[0], lo[1]);
}

template<bool BF16>
__device__ __forceinline__ uint4 encode16(const uint4* v, BlockScale s, bool redo)
{
    const uint2 a = encode8<BF16>(v[0], s, redo), b = encode8<BF16>(v[1], s, redo);
    return make_uint4(a.x, a.y, b.x, b.y);
}

// Blocks of 1 x 128.  A thread block takes 8 rows (one per warp) x 8 blocks of columns: eight lanes hold a block (two 16-byte
// loads each), a warp has 2 KB in flight, and the 64 scales go out through shared memory as runs of eight consecutive tokens.
template<bool BF16>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const uint4* __restrict__ x, uint4* __restrict__ codes, float* __restrict__ scales, int rows, int cols, int kb)
{
    __shared__ float tile[8][9];
    const int        warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int        kb_groups = (kb + 7) / 8;
    const int        row0      = static_cast<int>(blockIdx.x / kb_groups) * 8;
    const int        row       = row0 + warp;
    const int        kb0       = static_cast<int>(blockIdx.x % kb_groups) * 8;
    const int        per_row   = cols / 16;  // lanes' worth of elements
    const int        first     = kb0 * (kBlock / 16) + lane;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    if (row < rows) {
        const size_t base = static_cast<size_t>(row) * per_row + first;
        uint4        v[2][2];  // blocks kb0 + lane / 8 and that + 4
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                v[i][h] = first + 32 * i < per_row ? ptx::ld_once_128(x + 2 * (base + 32 * i) + h) : make_uint4(0, 0, 0, 0);
        // amax of the lane's two blocks, one per half of a register
        auto amax_of = [&](bool only_finite) {
            uint32_t m[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[i] = only_finite ? amax_bits(amax_bits(0u, finite_only<BF16>(v[i][0])), finite_only<BF16>(v[i][1]))
                                   : amax_bits(amax_bits(0u, v[i][0]), v[i][1]);
                m[i] = max(m[i] & 0xffffu, m[i] >> 16);
            }
            uint32_t pair = m[0] | (m[1] << 16);
#pragma unroll
            for (int d = 4; d > 0; d >>= 1)
                pair = __vmaxu2(pair, __shfl_xor_sync(0xffffffffu, pair, d));
            return pair;
        };
        uint32_t   pair = amax_of(false);
        const bool redo = __any_sync(0xffffffffu, max(pair & 0xffffu, pair >> 16) >= (kInfPair<BF16> & 0xffffu));
        if (redo)
            pair = amax_of(true);
        // even lanes work out the first block's scale, odd ones the second's
        const float scale = scale_of<BF16>((lane & 1) ? pair >> 16 : pair & 0xffffu);
        const BlockScale mine = block_scale(scale);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const BlockScale s{__shfl_sync(0xffffffffu, mine.scale, i, 8), __shfl_sync(0xffffffffu, mine.below, i, 8),
                               __shfl_sync(0xffffffffu, mine.above, i, 8)};
            if (first + 32 * i < per_row)
                codes[base + 32 * i] = encode16<BF16>(v[i], s, redo);
        }
        if ((lane & 7) < 2)
            tile[4 * (lane & 1) + (lane >> 3)][warp] = scale;
    }
    __syncthreads();
    const int k = threadIdx.x >> 3, r = threadIdx.x & 7;
    if (threadIdx.x < 64 && kb0 + k < kb && row0 + r < rows)
        scales[static_cast<size_t>(kb0 + k) * rows + row0 + r] = tile[k][r];
}

// Blocks of 128 x 128, one per thread block: 8 lanes per row, 32 rows per pass, the whole block (32 KB) in registers
// between the one read and the one write.  Four of them per SM: with two (the registers the compiler would take) the loads of
// one do not cover the arithmetic of the other (9208 x 36864, in a graph: 233 us, 179 with three, 156 with four, 219 with five,
// which spills).
template<bool BF16>
__global__ void __launch_bounds__(256, 4)
quantize_blocks_kernel(const uint4* __restrict__ x, uint4* __restrict__ codes, float* __restrict__ scales, int rows, int cols, int kb,
                       int row_blocks)
{
    __shared__ uint32_t warp_max[8];
    const int           kblock = static_cast<int>(blockIdx.x % kb);
    const int           rblock = static_cast<int>(blockIdx.x / kb) % row_blocks;
    const size_t        group  = blockIdx.x / (static_cast<unsigned>(kb) * row_blocks);
    const int           col    = kblock * (kBlock / 16) + (threadIdx.x & 7);
    const int           row0   = rblock * kBlock + static_cast<int>(threadIdx.x >> 3);
    const int           per_row = cols / 16;
    const size_t        base    = (group * rows + row0) * per_row + col;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    uint4 v[4][2];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
            v[i][h] = col < per_row && row0 + 32 * i < rows ? ptx::ld_once_128(x + 2 * (base + static_cast<size_t>(32 * i) * per_row) + h)
                                                            : make_uint4(0, 0, 0, 0);
    auto amax_of = [&](bool only_finite) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
            m = amax_bits(m, only_finite ? finite_only<BF16>(v[i / 2][i % 2]) : v[i / 2][i % 2]);
        m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
        if ((threadIdx.x & 31) == 0)
            warp_max[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++)
            m = max(m, warp_max[w]);
        return m;
    };
    uint32_t   m    = amax_of(false);
    const bool redo = m >= (kInfPair<BF16> & 0xffffu);
    if (redo) {
        __syncthreads();
        m = amax_of(true);
    }
    const BlockScale s = block_scale(scale_of<BF16>(m));
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (col < per_row && row0 + 32 * i < rows)
            codes[base + static_cast<size_t>(32 * i) * per_row] = encode16<BF16>(v[i], s, redo);
    if (threadIdx.x == 0)
        scales[blockIdx.x] = s.scale;
}

template<typename... P, typename... Args>
cudaError_t launch(cudaStream_t stream, void (*kern)(P...), dim3 grid, Args... args)
{
    cudaLaunchConfig_t config = {};
    config.gridDim            = grid;
    config.blockDim           = dim3(256);
    config.stream             = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs                                       = attr;
    config.numAttrs                                    = 1;
    cudaError_t e = cudaLaunchKernelEx(&config, kern, args...);
    if (e != cudaSuccess)
        (void)cudaGetLastError();
    return e;  // not what an earlier call has left behind
}

}  // namespace
}  // namespace spmm_b200

extern "C" int spmm_b200_quantize_fp8(
    void* stream, const void* X, int X_type, int groups, int rows, int cols, int block_rows, void* codes, float* scales)
{
    using namespace spmm_b200;
    if ((X_type != SPMM_B200_FP16 && X_type != SPMM_B200_BF16) || groups < 1 || rows < 0 || cols < 1 || cols % 16 != 0
        || (block_rows != 1 && block_rows != kBlock) || (block_rows == 1 && groups != 1))
        return static_cast<int>(cudaErrorInvalidValue);
    if (rows == 0)
        return static_cast<int>(cudaSuccess);
    if (!X || !codes || !scales || (reinterpret_cast<uintptr_t>(X) & 15u) || (reinterpret_cast<uintptr_t>(codes) & 15u)
        || (reinterpret_cast<uintptr_t>(scales) & 3u))
        return static_cast<int>(cudaErrorInvalidValue);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int    kb = (cols - 1) / kBlock + 1;
    if (block_rows == 1) {
        const long blocks = static_cast<long>((rows - 1) / 8 + 1) * ((kb - 1) / 8 + 1);
        if (blocks > 0x7fffffffL)
            return static_cast<int>(cudaErrorInvalidValue);
        auto kern = X_type == SPMM_B200_BF16 ? quantize_rows_kernel<true> : quantize_rows_kernel<false>;
        return static_cast<int>(launch(st, kern, dim3(static_cast<unsigned>(blocks)), static_cast<const uint4*>(X),
                                       static_cast<uint4*>(codes), scales, rows, cols, kb));
    }
    const int  row_blocks = (rows - 1) / kBlock + 1;
    const long blocks     = static_cast<long>(groups) * row_blocks * kb;
    if (blocks > 0x7fffffffL)
        return static_cast<int>(cudaErrorInvalidValue);
    auto kern = X_type == SPMM_B200_BF16 ? quantize_blocks_kernel<true> : quantize_blocks_kernel<false>;
    return static_cast<int>(launch(st, kern, dim3(static_cast<unsigned>(blocks)), static_cast<const uint4*>(X),
                                   static_cast<uint4*>(codes), scales, rows, cols, kb, row_blocks));
}
