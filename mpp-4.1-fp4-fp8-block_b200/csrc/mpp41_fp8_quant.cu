// Quantizers in front of the FP8 products: activations with a scale per 1 x 128
// and weights with a scale per 128 x 128 (amax / qmax, qmax = 448 for E4M3 and
// 57344 for E5M2; 1 where a block is all zero). Both read each value once, keep
// it in registers for the block's maximum, and write it back as 8 bits: bound by
// memory (3 or 5 bytes a value; 4096 x 7168 activations in 15.3 us, 88 % of the copy rate).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "mpp41_device.cuh"
#include "mpp41_fp8.cuh"
#include "mpp41_internal.h"

namespace mpp41 {
namespace fp8 {

constexpr uint32_t kBlock = 128;

constexpr uint32_t blocks_of(uint32_t n) { return n / kBlock + (n % kBlock != 0); }   // of any n: no sum that wraps

// 16 fp16 values a lane, 8 lanes a block: rows of H % 16 == 0 values, x 32-byte
// and q 16-byte aligned. A block behind the row's end is short in its last lanes.
template <int FMT>
__global__ void __launch_bounds__(256) quant_act_kernel(const uint8_t *__restrict__ x, uint32_t H, uint32_t kb,
                                                        uint64_t blocks, uint8_t *__restrict__ q, float *__restrict__ scales)
{
    pdl_wait_prior();
    const uint32_t sub = threadIdx.x & 7;
    const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 8);
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x / 8) + threadIdx.x / 8; __any_sync(0xffffffffu, i < blocks); i += step) {
        const uint64_t t = i / kb;
        const uint32_t c = (uint32_t)(i - t * kb) * kBlock + sub * 16;
        const bool have = i < blocks && c < H;
        const uint64_t at = t * H + c;
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0u;
        if (have) load_act16(x + at * 2, w);
        float scale;
        const uint4 o = quant_act16<FMT>(w, scale);
        if (have) *reinterpret_cast<uint4 *>(q + at) = o;
        if (i < blocks && sub == 0) scales[i] = scale;
    }
}

// Any width and alignment: one warp a block, four values a lane.
template <int FMT>
__global__ void __launch_bounds__(256) quant_act_any_kernel(const __half *__restrict__ x, uint32_t H, uint32_t kb,
                                                            uint64_t blocks, uint8_t *__restrict__ q, float *__restrict__ scales)
{
    pdl_wait_prior();
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 32);
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; i < blocks; i += step) {
        const uint64_t t = i / kb;
        const uint32_t c = (uint32_t)(i - t * kb) * kBlock + lane;
        const __half *row = x + t * H;
        float v[4], amax = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            v[j] = c + 32 * j < H ? __half2float(row[c + 32 * j]) : 0.0f;
            amax = fmaxf(amax, fabsf(v[j]));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        amax = amax_h(amax);
        float mul, scale;
        block_scale(amax, f8_max(FMT), mul, scale);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (c + 32 * j < H) q[t * H + c + 32 * j] = (uint8_t)enc_f8x2(FMT, snap(v[j], mul), 0.0f);
        if (lane == 0) scales[i] = scale;
    }
}

// round(w * qmax / amax), exactly: 7 w and m * amax, m a midpoint of the
// 8-bit format (5 bits), are integers of 27 and 29 bits, so the quotient is a midpoint or at
// least 2^-30 of its size away from one, which 64 bits tell apart. The quotient reaches the
// encoder as fp32 cut to zero, its lowest bit set where anything was cut: a value next to a
// midpoint stays on its side.
template <int FMT> __device__ __forceinline__ uint8_t exact_f8(float w, float amax)
{
    const double d = (double)w * (double)f8_max(FMT) / (double)amax;
    float f = __double2float_rz(d);
    if ((double)f != d) f = __uint_as_float(__float_as_uint(f) | 1u);
    return (uint8_t)enc_f8x2(FMT, f, 0.0f);
}

// One CTA a 128 x 128 block, 32 fp32 values a thread (two CTAs an SM, so that one's loads
// cover another's stores): warp w has rows w, w + 16, ..., a lane four neighbouring columns
// (VEC: K % 4 == 0 and aligned pointers).
// q = round(w * qmax / amax), correctly rounded: fp32 products with a factor 2^-21 below and
// one as far above the quotient, which their three roundings (2^-24 each) do not bridge. Where
// both give the same code it is the exact quotient's, elsewhere (one value in 10^5) 64 bits
// decide: 14336 x 4096 in 48.3 us, 93 % of the copy rate (48.0 with one rounded factor and
// wrong codes at some midpoints, 57 with a division a value).
template <int FMT, bool VEC>
__global__ void __launch_bounds__(512, 2) quant_weights_kernel(const float *__restrict__ w, uint32_t N, uint32_t K, uint32_t kb,
                                                            uint8_t *__restrict__ q, float *__restrict__ scales)
{
    __shared__ float part[16];
    pdl_wait_prior();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t bn = blockIdx.x / kb, bk = blockIdx.x - bn * kb;
    const uint32_t c = bk * kBlock + 4 * lane;
    float4 v[8];
    float amax = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t r = bn * kBlock + warp + 16 * j;
        const float *src = w + (size_t)r * K + c;
        v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < N) {
            if (VEC) {
                if (c < K) v[j] = __ldcs(reinterpret_cast<const float4 *>(src));
            } else {
                if (c < K) v[j].x = src[0];
                if (c + 1 < K) v[j].y = src[1];
                if (c + 2 < K) v[j].z = src[2];
                if (c + 3 < K) v[j].w = src[3];
            }
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(v[j].x), fabsf(v[j].y))), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) part[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = fmaxf(amax, part[j]);
    amax = fminf(amax, 3.402823466e38f);   // infinity counts as the largest finite value
    const float by = amax > 0.0f ? amax : 1.0f, qmax = f8_max(FMT);
    // qmax / amax would overflow for the smallest maxima: those blocks are raised first, which is exact
    const float raise = by < 0x1p-100f ? 0x1p100f : 1.0f, mul = __fdiv_rn(qmax, by * raise);
    const float below = mul * (1.0f - 0x1p-21f), above = mul * (1.0f + 0x1p-21f);
    if (threadIdx.x == 0) scales[blockIdx.x] = amax > 0.0f ? __fdiv_rn(amax, qmax) : 1.0f;
    uint32_t open = 0;   // bit j: a code of v[j] is not settled
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t r = bn * kBlock + warp + 16 * j;
        if (r >= N || c >= K) continue;
        const float4 u = make_float4(v[j].x * raise, v[j].y * raise, v[j].z * raise, v[j].w * raise);
        const uint32_t o = enc_f8x2(FMT, u.x * below, u.y * below) | enc_f8x2(FMT, u.z * below, u.w * below) << 16;
        const uint32_t o1 = enc_f8x2(FMT, u.x * above, u.y * above) | enc_f8x2(FMT, u.z * above, u.w * above) << 16;
        if (o != o1) open |= 1u << j;
        uint8_t *dst = q + (size_t)r * K + c;
        if (VEC) {
            *reinterpret_cast<uint32_t *>(dst) = o;
        } else {
            dst[0] = (uint8_t)o;
            if (c + 1 < K) dst[1] = (uint8_t)(o >> 8);
            if (c + 2 < K) dst[2] = (uint8_t)(o >> 16);
            if (c + 3 < K) dst[3] = (uint8_t)(o >> 24);
        }
    }
    // the few open ones read their values again: kept until here they would cost the others registers
    for (; open; open &= open - 1) {
        const size_t at = (size_t)(bn * kBlock + warp + 16 * (__ffs(open) - 1)) * K + c;
        for (uint32_t i = 0; i < 4 && c + i < K; ++i) q[at + i] = exact_f8<FMT>(w[at + i], by);
    }
}

}  // namespace fp8

cudaError_t launch_quantize_act_fp8(int fmt, const void *x, uint32_t T, uint32_t H, uint8_t *q, float *scales, cudaStream_t st)
{
    using namespace fp8;
    const uint32_t kb = blocks_of(H);
    const uint64_t blocks = (uint64_t)T * kb;
    if (!blocks) return cudaSuccess;
    const bool wide = H % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 31u) == 0 && (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
    const uint64_t per = wide ? 32 : 8, need = (blocks + per - 1) / per;
    const unsigned grid = (unsigned)(need < 148 * 16 ? need : 148 * 16);
    const uint8_t *xb = static_cast<const uint8_t *>(x);
    const __half *xh = static_cast<const __half *>(x);
    if (wide)
        return launch_overlapped(fmt == 1 ? quant_act_kernel<1> : quant_act_kernel<2>, dim3(grid), dim3(256), 0, st, xb, H, kb, blocks, q, scales);
    return launch_overlapped(fmt == 1 ? quant_act_any_kernel<1> : quant_act_any_kernel<2>, dim3(grid), dim3(256), 0, st, xh, H, kb, blocks, q, scales);
}

cudaError_t launch_quantize_weights_fp8(int fmt, const float *w, uint32_t N, uint32_t K, uint8_t *q, float *scales, cudaStream_t st)
{
    using namespace fp8;
    if (!N || !K) return cudaSuccess;
    const uint32_t kb = blocks_of(K), nb = blocks_of(N);
    const bool vec = K % 4 == 0 && (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && (reinterpret_cast<uintptr_t>(q) & 3u) == 0;
    const unsigned grid = nb * kb;   // the caller keeps it below 2^31
    return launch_overlapped(vec ? (fmt == 1 ? quant_weights_kernel<1, true> : quant_weights_kernel<2, true>)
                                 : (fmt == 1 ? quant_weights_kernel<1, false> : quant_weights_kernel<2, false>),
                             dim3(grid), dim3(512), 0, st, w, N, K, kb, q, scales);
}

}  // namespace mpp41
