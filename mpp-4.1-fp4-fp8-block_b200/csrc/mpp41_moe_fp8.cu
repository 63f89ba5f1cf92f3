// The pieces of the FP8 expert layer around its two grouped products
// (mpp41_fp8_gemm.cuh), for T tokens, k assignments a token, E experts:
//   plan:     ids [T][k] -> offsets[E+1] (rows of each expert) and inv[T*k]
//             (assignment -> row, -1 where the id names no expert). Rows are grouped
//             by expert and keep assignment order inside one: deterministic.
//   scatter:  x is quantized once (1 x 128 scales) and each block written to the
//             rows of its token's assignments; no gather pass reads it again.
//   experts:  grouped gate/up product with the SwiGLU + quantization epilogue, then
//             the grouped down product, each row times its routing weight
//             -> y [rows][H]; the shared expert's tiles run in the same two launches.
//   combine:  out[t] = shared(t) + sum_j y[inv[t*k+j]], in slot order, summed in fp32.
// y and the shared expert's rows are fp32 whatever out's type: terms of opposite sign may
// cancel, and two of more than 65504 leave a finite sum that fp16 rows would lose. An fp16
// out is rounded once, from the sum. (fp16 rows: 1020 against 1093 us for 2048 tokens of
// the 7168 / 2048 layer, 8 of 32 experts; no difference for one token.)
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "mpp41_device.cuh"
#include "mpp41_fp8.cuh"
#include "mpp41_internal.h"

namespace mpp41 {
namespace fp8 {

constexpr int kPlanThreads = 512;

// Rows of expert e: one CTA reading all ids twice (they sit in L2): rows before e's = ids
// below it, then a stable compaction. A warp owns a contiguous run of assignments, read in
// chunks of 32 x 4, so one sum over the warps orders them; inside a chunk, which seldom
// holds one of e's, lanes are ordered by a scan. No launch or wait joins the experts' CTAs.
template <int THREADS>
__device__ __forceinline__ void plan_expert(const int32_t *__restrict__ ids, const float *__restrict__ weights, uint32_t n, uint32_t E,
                                            int32_t e, int32_t *__restrict__ offsets, int32_t *__restrict__ inv,
                                            float *__restrict__ row_weight, uint32_t *err)
{
    constexpr uint32_t kWarps = THREADS / 32;
    __shared__ uint32_t sh_lt[kWarps], sh_eq[kWarps];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t chunks = (n + 127) / 128, per = (chunks + kWarps - 1) / kWarps;
    const uint32_t c0 = min(warp * per, chunks), c1 = min(c0 + per, chunks);
    const bool vec = (reinterpret_cast<uintptr_t>(ids) & 15u) == 0;
    auto load = [&](uint32_t c) {                       // this lane's four ids of a chunk, -1 behind the last
        const uint32_t a = c * 128 + lane * 4;
        if (vec && a + 4 <= n) return *reinterpret_cast<const int4 *>(ids + a);
        return make_int4(a < n ? ids[a] : -1, a + 1 < n ? ids[a + 1] : -1, a + 2 < n ? ids[a + 2] : -1, a + 3 < n ? ids[a + 3] : -1);
    };
    auto equal = [&](const int4 &v) { return (v.x == e ? 1u : 0u) | (v.y == e ? 2u : 0u) | (v.z == e ? 4u : 0u) | (v.w == e ? 8u : 0u); };
    uint32_t lt = 0, eq = 0;
    bool bad = false;
#pragma unroll 4
    for (uint32_t c = c0; c < c1; ++c) {
        const int4 v = load(c);
        // unsigned: an id below 0 is above every expert
        lt += ((uint32_t)v.x < (uint32_t)e) + ((uint32_t)v.y < (uint32_t)e) + ((uint32_t)v.z < (uint32_t)e) + ((uint32_t)v.w < (uint32_t)e);
        eq += __popc(equal(v));
        if (e == 0) {
            const int32_t id[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t a = c * 128 + lane * 4 + j;
                if (a < n && (uint32_t)id[j] >= E) {
                    inv[a] = -1;
                    bad |= id[j] >= 0;
                }
            }
        }
    }
    if (bad) report_error(err, kErrBounds, 0xF91);
    lt = __reduce_add_sync(0xffffffffu, lt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        sh_lt[warp] = lt;
        sh_eq[warp] = eq;
    }
    __syncthreads();
    uint32_t base = 0, all = 0, before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        base += sh_lt[w];
        all += sh_eq[w];
        before += w < warp ? sh_eq[w] : 0u;
    }
    if (threadIdx.x == 0) {
        offsets[e] = (int32_t)base;
        if (e == (int32_t)E - 1) offsets[E] = (int32_t)(base + all);
    }
    uint32_t row = base + before;
    const uint32_t last = row + eq;
    for (uint32_t c = c0; c < c1 && row < last; ++c) {
        const uint32_t m = equal(load(c)), mine = __popc(m);
        if (!__any_sync(0xffffffffu, m != 0)) continue;
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += v;
        }
        uint32_t r = row + inc - mine;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (m >> j & 1u) {
                const uint32_t a = c * 128 + lane * 4 + j;
                row_weight[r] = weights[a];
                inv[a] = (int32_t)r++;
            }
        row += __shfl_sync(0xffffffffu, inc, 31);
    }
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t *__restrict__ ids, const float *__restrict__ weights,
                                                            uint32_t n, uint32_t E, int32_t *__restrict__ offsets,
                                                            int32_t *__restrict__ inv, float *__restrict__ row_weight, uint32_t *err)
{
    plan_expert<kPlanThreads>(ids, weights, n, E, (int32_t)blockIdx.x, offsets, inv, row_weight, err);
}

// As the activation quantizer (8 lanes a block of 128, 16 values a lane), each block
// written to the rows inv[t*k + j] >= 0 and, where xq is given, to row t of xq.
template <int FMT>
__global__ void __launch_bounds__(256) quant_scatter_kernel(const uint8_t *__restrict__ x, uint32_t kb, uint64_t blocks,
                                                            const int32_t *__restrict__ inv, uint32_t k,
                                                            uint8_t *__restrict__ pq, float *__restrict__ ps,
                                                            uint8_t *__restrict__ xq, float *__restrict__ xs)
{
    const uint32_t sub = threadIdx.x & 7;
    const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 8);
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x / 8) + threadIdx.x / 8; __any_sync(0xffffffffu, i < blocks); i += step) {
        const bool have = i < blocks;
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0u;
        if (have) load_act16(x + (i * 128 + sub * 16) * 2, w);
        float scale;
        const uint4 o = quant_act16<FMT>(w, scale);
        if (!have) continue;
        const uint64_t t = i / kb;
        const uint32_t b = (uint32_t)(i - t * kb);
        if (xq) {
            *reinterpret_cast<uint4 *>(xq + i * 128 + sub * 16) = o;
            if (sub == 0) xs[i] = scale;
        }
        for (uint32_t j = 0; j < k; ++j) {
            const int32_t r = inv[t * k + j];
            if (r < 0) continue;
            const uint64_t at = (uint64_t)r * kb + b;
            *reinterpret_cast<uint4 *>(pq + at * 128 + sub * 16) = o;
            if (sub == 0) ps[at] = scale;
        }
    }
}

// Plan and scatter in one launch, for few assignments: the first E CTAs plan, the others
// scatter 32 blocks each and count the rows of their tokens' assignments themselves (ids
// below theirs, and equal ones before theirs: a warp an assignment over all n ids).
constexpr uint32_t kFewIds = 2048;       // ids kept in shared memory
constexpr uint32_t kFewRows = 256;       // assignments a CTA counts for

template <int FMT>
__global__ void __launch_bounds__(256) plan_scatter_kernel(const int32_t *__restrict__ ids, const float *__restrict__ weights,
                                                           uint32_t n, uint32_t E, int32_t *__restrict__ offsets,
                                                           int32_t *__restrict__ inv, float *__restrict__ row_weight, uint32_t *err,
                                                           const uint8_t *__restrict__ x, uint32_t kb, uint32_t blocks, uint32_t k,
                                                           uint8_t *__restrict__ pq, float *__restrict__ ps,
                                                           uint8_t *__restrict__ xq, float *__restrict__ xs)
{
    __shared__ int32_t sh_ids[kFewIds];
    __shared__ int32_t rows[kFewRows];
    if (blockIdx.x < E) {
        plan_expert<256>(ids, weights, n, E, (int32_t)blockIdx.x, offsets, inv, row_weight, err);
        return;
    }
    const uint32_t i0 = (blockIdx.x - E) * 32, i = i0 + threadIdx.x / 8, sub = threadIdx.x & 7;
    const bool have = i < blocks;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 0u;
    if (have) load_act16(x + ((size_t)i * 128 + sub * 16) * 2, w);
    for (uint32_t a = threadIdx.x; a < n; a += 256) sh_ids[a] = ids[a];
    __syncthreads();
    const uint32_t t0 = i0 / kb, t1 = min(i0 + 31, blocks - 1) / kb, first = t0 * k, count = (t1 - t0 + 1) * k;
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t q = threadIdx.x >> 5; q < count; q += 8) {
        const int32_t e = sh_ids[first + q];
        uint32_t c = 0;
        for (uint32_t a = lane; a < n; a += 32) {
            const int32_t id = sh_ids[a];
            c += id >= 0 && (id < e || (id == e && a < first + q)) ? 1u : 0u;
        }
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) rows[q] = e >= 0 && e < (int32_t)E ? (int32_t)c : -1;
    }
    __syncthreads();
    float scale;
    const uint4 o = quant_act16<FMT>(w, scale);
    if (!have) return;
    const uint32_t t = i / kb, b = i - t * kb;
    if (xq) {
        *reinterpret_cast<uint4 *>(xq + (size_t)i * 128 + sub * 16) = o;
        if (sub == 0) xs[i] = scale;
    }
    for (uint32_t j = 0; j < k; ++j) {
        const int32_t r = rows[(t - t0) * k + j];
        if (r < 0) continue;
        const size_t at = (size_t)r * kb + b;
        *reinterpret_cast<uint4 *>(pq + at * 128 + sub * 16) = o;
        if (sub == 0) ps[at] = scale;
    }
}

// One CTA per token and 128 units of 16 bytes (the grid's limit only makes it go on to
// others); slots summed in order, fp32. A thread has eight rows' loads in flight: with one
// token that is the whole kernel.
constexpr int kCombineThreads = 128;

template <bool F16>
__global__ void __launch_bounds__(kCombineThreads) combine_fp8_kernel(const float4 *__restrict__ y, const int32_t *__restrict__ inv,
                                                                      uint32_t k, uint32_t units,
                                                                      const float4 *__restrict__ shared_y, void *__restrict__ out)
{
    __shared__ int32_t rows[32];
    const uint32_t t = blockIdx.x;
    if (threadIdx.x < k) rows[threadIdx.x] = inv[(size_t)t * k + threadIdx.x];
    uint32_t c = blockIdx.y * kCombineThreads + threadIdx.x;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (shared_y && c < units) acc = __ldcs(shared_y + (size_t)t * units + c);
    __syncthreads();
    while (c < units) {
        for (uint32_t j0 = 0; j0 < k; j0 += 8) {
            float4 v[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                const int32_t r = j0 + j < k ? rows[j0 + j] : -1;
                v[j] = r >= 0 ? __ldcs(y + (size_t)r * units + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                acc.x += v[j].x;
                acc.y += v[j].y;
                acc.z += v[j].z;
                acc.w += v[j].w;
            }
        }
        const size_t at = (size_t)t * units + c;
        if (F16) static_cast<uint2 *>(out)[at] = make_uint2(half2_bits(acc.x, acc.y), half2_bits(acc.z, acc.w));
        else static_cast<float4 *>(out)[at] = acc;
        c += gridDim.y * kCombineThreads;
        acc = shared_y && c < units ? __ldcs(shared_y + (size_t)t * units + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
}

}  // namespace fp8

cudaError_t launch_fp8_scatter(int fmt, const int32_t *ids, const float *weights, uint32_t E, int32_t *offsets, int32_t *inv,
                               float *row_weight, uint32_t *err, const void *x, uint32_t T, uint32_t H, uint32_t k, uint8_t *pq,
                               float *ps, uint8_t *xq, float *xs, cudaStream_t st)
{
    using namespace fp8;
    const uint32_t n = T * k, kb = H / 128;
    const uint64_t blocks = (uint64_t)T * kb, need = (blocks + 31) / 32;
    const uint8_t *xb = static_cast<const uint8_t *>(x);
    // one launch (3 us less) where counting stays short: a CTA's assignments times all ids
    const uint64_t mine = (31 / kb + 2) * (uint64_t)k;
    if (n <= kFewIds && mine <= kFewRows && mine * n <= 32768) {
        const unsigned grid = E + (unsigned)need;
        if (fmt == 1)
            plan_scatter_kernel<1><<<grid, 256, 0, st>>>(ids, weights, n, E, offsets, inv, row_weight, err, xb, kb, (uint32_t)blocks, k, pq, ps, xq, xs);
        else
            plan_scatter_kernel<2><<<grid, 256, 0, st>>>(ids, weights, n, E, offsets, inv, row_weight, err, xb, kb, (uint32_t)blocks, k, pq, ps, xq, xs);
        return cudaGetLastError();
    }
    plan_kernel<<<E, kPlanThreads, 0, st>>>(ids, weights, n, E, offsets, inv, row_weight, err);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned)(need < 148 * 16 ? need : 148 * 16);
    if (fmt == 1) quant_scatter_kernel<1><<<grid, 256, 0, st>>>(xb, kb, blocks, inv, k, pq, ps, xq, xs);
    else quant_scatter_kernel<2><<<grid, 256, 0, st>>>(xb, kb, blocks, inv, k, pq, ps, xq, xs);
    return cudaGetLastError();
}

cudaError_t launch_fp8_combine(const float *y, const int32_t *inv, uint32_t T, uint32_t k, uint32_t H, const float *shared_y,
                               void *out, int f16, cudaStream_t st)
{
    const uint32_t units = H / 4, chunks = (units + fp8::kCombineThreads - 1) / fp8::kCombineThreads;
    const dim3 grid(T, chunks < 65535 ? chunks : 65535);
    const float4 *a = reinterpret_cast<const float4 *>(y), *sy = reinterpret_cast<const float4 *>(shared_y);
    if (f16) fp8::combine_fp8_kernel<true><<<grid, fp8::kCombineThreads, 0, st>>>(a, inv, k, units, sy, out);
    else fp8::combine_fp8_kernel<false><<<grid, fp8::kCombineThreads, 0, st>>>(a, inv, k, units, sy, out);
    return cudaGetLastError();
}

}  // namespace mpp41
