// 8-bit floating point encoding and the activation quantizer's arithmetic, shared by
// the FP8 quantizers, the expert layer's scatter and the GEMM epilogue.
#pragma once

#include <cuda_fp16.h>
#include <cstdint>

namespace mpp41 {
namespace fp8 {

// fmt 1 = E4M3, 2 = E5M2 (the format numbers of mpp41_pack).
__host__ __device__ constexpr float f8_max(int fmt) { return fmt == 1 ? 448.0f : 57344.0f; }

// Two values to 8 bits, round to nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t enc_f8x2(int fmt, float lo, float hi)
{
    uint16_t r;
    if (fmt == 1)
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// |x| as the maximum sees it: NaN counts as nothing, infinity as the largest finite fp16.
__device__ __forceinline__ float amax_h(float amax) { return fminf(amax, 65504.0f); }

// Multiplier and scale of a block. q = round(x * qmax / amax) has to be exact: x
// and amax are 11-bit numbers and qmax = 7 * 2^n, so x * qmax / amax either is a
// midpoint of the 8-bit format (at most 5 significant bits) or is at least 2^-16
// of its size away from one. The product with the rounded quotient qmax / amax is
// within 2^-22; raising it by 0.7 * 2^-20 and cutting it to 20 significant bits
// (snap) puts it on the midpoint in the first case and leaves its side alone in
// the second, for one multiplication and one AND instead of a division a value.
__device__ __forceinline__ void block_scale(float amax, float qmax, float &mul, float &scale)
{
    mul = amax > 0.0f ? __fmul_rn(__fdiv_rn(qmax, amax), 1.0f + 0.7f / 1048576.0f) : 0.0f;
    scale = amax > 0.0f ? __fdiv_rn(amax, qmax) : 1.0f;
}

__device__ __forceinline__ float snap(float x, float mul)
{
    return __uint_as_float(__float_as_uint(x * mul) & ~15u);
}

// 16 fp16 values, 32-byte aligned.
__device__ __forceinline__ void load_act16(const uint8_t *p, uint32_t (&w)[8])
{
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}

// One lane's 16 values of a block held by 8 neighbouring lanes (all 32 lanes call it).
template <int FMT> __device__ __forceinline__ uint4 quant_act16(const uint32_t (&w)[8], float &scale)
{
    auto h2 = [&](int j) { return *reinterpret_cast<const __half2 *>(&w[j]); };
    __half2 m2 = __habs2(h2(0));
#pragma unroll
    for (int j = 1; j < 8; ++j) m2 = __hmax2(m2, __habs2(h2(j)));
    float amax = fmaxf(__low2float(m2), __high2float(m2));
#pragma unroll
    for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    amax = amax_h(fmaxf(amax, 0.0f));   // fmaxf: NaN -> 0
    float mul;
    block_scale(amax, f8_max(FMT), mul, scale);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 a = __half22float2(h2(2 * j)), b = __half22float2(h2(2 * j + 1));
        o[j] = enc_f8x2(FMT, snap(a.x, mul), snap(a.y, mul)) | enc_f8x2(FMT, snap(b.x, mul), snap(b.y, mul)) << 16;
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace fp8
}  // namespace mpp41
