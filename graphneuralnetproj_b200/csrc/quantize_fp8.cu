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
// Rounding to the nearest value of the *exact* quotient: x * (1 / s) is off by at most two units in the last place of
// fp32, so the rounding of that product can differ from the rounding of the quotient only where the product lies within
// a few units of the midpoint between two e4m3 values.  Those elements (about one in 10^5) take the slow path: the
// correctly rounded quotient, and where the remainder is not zero a step of one unit towards the exact quotient if that
// makes the last bit odd -- a midpoint is a number of five bits and never odd, so the second rounding then sees the right
// side.
//
// Bound by memory (2 bytes in, 1 out per element) once an element costs about ten instructions.  Dividing every element,
// or sending the ones below the smallest normal e4m3 value down the slow path (a few per cent of them where some features
// are much larger than others, so nearly every warp), made it twice as slow.
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

__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi)
{
    uint16_t out;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(hi), "f"(lo));
    return out;
}

// The quotient x / s as an fp32 number that rounds to e4m3 as the exact quotient does.
__device__ __forceinline__ float quotient_for_rounding(float x, float s)
{
    const float q = __fdiv_rn(x, s);
    if (!(fabsf(x) <= 3.4028234663852886e38f))
        return __int_as_float(0x7fffffff);  // infinite or NaN
    const float r = __fmaf_rn(-q, s, x);  // exact
    int         b = __float_as_int(q);
    if (r != 0.0f && (b & 1) == 0)
        b += ((__float_as_int(r) ^ b) >= 0) ? 1 : -1;
    return __int_as_float(b);
}

// Whether the rounding of y, an approximation of the quotient within two units in the last place, may differ from the
// rounding of the quotient itself: y is within four units of a midpoint, i.e. its 20 bits below those e4m3 keeps are near
// 10...0.  Below 2^-6 e4m3 is evenly spaced, as fp32 is between 2^-6 and 2^-5 cut to three bits, so y is looked at there.
__device__ __forceinline__ bool doubtful(float y)
{
    float t = fabsf(y);
    t       = t < 0.015625f ? t + 0.015625f : t;
    return (__float_as_uint(t) << 12) - (0x7fffcu << 12) <= (8u << 12);
}

// Eight elements (one 16-byte load) to eight codes.  redo: the block holds elements that are not finite.
template<bool BF16>
__device__ __forceinline__ uint2 encode8(uint4 v, float s, float inv, bool redo)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float          y[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[2 * i]     = element<BF16>(w[i] & 0xffffu) * inv;
        y[2 * i + 1] = element<BF16>(w[i] >> 16) * inv;
        redo |= doubtful(y[2 * i]) | doubtful(y[2 * i + 1]);
    }
    if (redo) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[2 * i]     = quotient_for_rounding(element<BF16>(w[i] & 0xffffu), s);
            y[2 * i + 1] = quotient_for_rounding(element<BF16>(w[i] >> 16), s);
        }
    }
    return make_uint2(e4m3_pair(y[0], y[1]) | (e4m3_pair(y[2], y[3]) << 16), e4m3_pair(y[4], y[5]) | (e4m3_pair(y[6], y[7]) << 16));
}

// Blocks of 1 x 128.  A thread block takes 8 rows (one per warp) x 8 blocks of columns: a half-warp holds a block (16
// bytes per lane), so a warp reads 512 contiguous bytes per load and has four of them in flight, and the 64 scales go
// out through shared memory as runs of eight consecutive tokens.
template<bool BF16>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const uint4* __restrict__ x, uint2* __restrict__ codes, float* __restrict__ scales, int rows, int cols, int kb)
{
    __shared__ float tile[8][9];
    const int        warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int        kb_groups = (kb + 7) / 8;
    const int        row0      = static_cast<int>(blockIdx.x / kb_groups) * 8;
    const int        row       = row0 + warp;
    const int        kb0       = static_cast<int>(blockIdx.x % kb_groups) * 8;
    const int        per_row   = cols / 8;
    const int        first     = kb0 * (kBlock / 8) + lane;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    if (row < rows) {
        const size_t base = static_cast<size_t>(row) * per_row;
        uint4        v[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = first + 32 * i < per_row ? ptx::ld_stream_128(x + base + first + 32 * i) : make_uint4(0, 0, 0, 0);
        // amax of this half-warp's four blocks, two blocks to a register
        auto amax_of = [&](bool only_finite, uint32_t* pair) {
            uint32_t m[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                m[i] = amax_bits(0u, only_finite ? finite_only<BF16>(v[i]) : v[i]);
                m[i] = max(m[i] & 0xffffu, m[i] >> 16);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                pair[i] = m[2 * i] | (m[2 * i + 1] << 16);
#pragma unroll
                for (int d = 8; d > 0; d >>= 1)
                    pair[i] = __vmaxu2(pair[i], __shfl_xor_sync(0xffffffffu, pair[i], d));
            }
        };
        uint32_t pair[2];
        amax_of(false, pair);
        const uint32_t most = __vmaxu2(pair[0], pair[1]);
        const bool     redo = __any_sync(0xffffffffu, max(most & 0xffffu, most >> 16) >= (kInfPair<BF16> & 0xffffu));
        if (redo)
            amax_of(true, pair);
        // lane i of a half computes block i's scale and its reciprocal for the others
        const uint32_t mine  = (lane & 2) ? pair[1] : pair[0];
        const float    scale = scale_of<BF16>((lane & 1) ? mine >> 16 : mine & 0xffffu);
        const float    recip = __frcp_rn(scale);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float s   = __shfl_sync(0xffffffffu, scale, i, 16);
            const float inv = __shfl_sync(0xffffffffu, recip, i, 16);
            if (first + 32 * i < per_row)
                codes[base + first + 32 * i] = encode8<BF16>(v[i], s, inv, redo);
        }
        if ((lane & 15) < 4)
            tile[2 * (lane & 3) + (lane >> 4)][warp] = scale;
    }
    __syncthreads();
    const int k = threadIdx.x >> 3, r = threadIdx.x & 7;
    if (threadIdx.x < 64 && kb0 + k < kb && row0 + r < rows)
        scales[static_cast<size_t>(kb0 + k) * rows + row0 + r] = tile[k][r];
}

// Blocks of 128 x 128, one per thread block: 16 lanes per row, 16 rows per pass, the whole block (32 KB) in registers
// between the one read and the one write.
template<bool BF16>
__global__ void __launch_bounds__(256)
quantize_blocks_kernel(const uint4* __restrict__ x, uint2* __restrict__ codes, float* __restrict__ scales, int rows, int cols, int kb,
                       int row_blocks)
{
    __shared__ uint32_t warp_max[8];
    const int           kblock = static_cast<int>(blockIdx.x % kb);
    const int           rblock = static_cast<int>(blockIdx.x / kb) % row_blocks;
    const size_t        group  = blockIdx.x / (static_cast<unsigned>(kb) * row_blocks);
    const int           col    = kblock * (kBlock / 8) + (threadIdx.x & 15);
    const int           row0   = rblock * kBlock + static_cast<int>(threadIdx.x >> 4);
    const int           per_row = cols / 8;
    const size_t        base    = group * rows * static_cast<size_t>(per_row) + col;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    uint4    v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        v[i] = col < per_row && row0 + 16 * i < rows ? ptx::ld_stream_128(x + base + static_cast<size_t>(row0 + 16 * i) * per_row)
                                                     : make_uint4(0, 0, 0, 0);
    auto amax_of = [&](bool only_finite) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
            m = amax_bits(m, only_finite ? finite_only<BF16>(v[i]) : v[i]);
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
    const float s   = scale_of<BF16>(m);
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (col < per_row && row0 + 16 * i < rows)
            codes[base + static_cast<size_t>(row0 + 16 * i) * per_row] = encode8<BF16>(v[i], s, inv, redo);
    if (threadIdx.x == 0)
        scales[blockIdx.x] = s;
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
    return e != cudaSuccess ? e : cudaGetLastError();
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
                                       static_cast<uint2*>(codes), scales, rows, cols, kb));
    }
    const int  row_blocks = (rows - 1) / kBlock + 1;
    const long blocks     = static_cast<long>(groups) * row_blocks * kb;
    if (blocks > 0x7fffffffL)
        return static_cast<int>(cudaErrorInvalidValue);
    auto kern = X_type == SPMM_B200_BF16 ? quantize_blocks_kernel<true> : quantize_blocks_kernel<false>;
    return static_cast<int>(launch(st, kern, dim3(static_cast<unsigned>(blocks)), static_cast<const uint4*>(X),
                                   static_cast<uint2*>(codes), scales, rows, cols, kb, row_blocks));
}
