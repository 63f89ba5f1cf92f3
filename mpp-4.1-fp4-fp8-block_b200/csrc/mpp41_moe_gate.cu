// Expert routing: scores (softmax or sigmoid), a balance bias that only the
// selection sees, expert groups, top-k and renormalised weights, one warp a token.
//
// Selection value of expert e: v = score + bias (-inf where the logit is -inf or
// NaN: a masked expert). With groups, a group's worth is the sum of its group_top
// largest v; the top_groups best groups stay, and the top_k experts are taken
// from them by falling v, ties to the lower index.
//
// The selection is exact: it is the one the 64-bit values give. Without a bias
// (and without sums of two scores) v is monotone in the logit, so the logits are
// compared themselves. Otherwise fp32 scores decide, and wherever two values that
// the outcome depends on lie closer than the fp32 error, that warp computes the
// token again in 64 bits: about one token in a thousand for scores of a trained
// router's spread, which costs less than 64-bit exponentials for all of them.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "mpp41_device.cuh"
#include "mpp41_internal.h"

namespace mpp41 {
namespace gate {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kWarps = 4;

struct Params {
    const void *logits;     // [T][E] fp32 or fp16
    const float *bias;      // [E] or null
    int32_t *ids;           // [T][k]
    float *weights;         // [T][k]
    uint32_t T, E, k, groups, top_groups, group_top, group_size;
    int sigmoid, renorm, f16, by_logit;   // by_logit: v is the logit
    float scale;
};

// fp32 fast exponentials: the scores' absolute error is below 2^-20 (a sigmoid's
// slope times the exponent's error peaks at 0.25 * 2^-20, a softmax value's at
// 0.37 * 2^-20 plus its sum's); sums with a bias add half an ulp of |v|.
constexpr float kTol = 1.0f / 524288.0f;

template <typename F> struct Num;
template <> struct Num<float> {
    static __device__ __forceinline__ float exp(float x) { return __expf(x); }
    static __device__ __forceinline__ float rcp(float x) { return __fdividef(1.0f, x); }
    static __device__ __forceinline__ float inf() { return INFINITY; }
};
template <> struct Num<double> {
    static __device__ __forceinline__ double exp(double x) { return ::exp(x); }
    static __device__ __forceinline__ double rcp(double x) { return 1.0 / x; }
    static __device__ __forceinline__ double inf() { return (double)INFINITY; }
};

__device__ __forceinline__ float load_logit(const Params &p, size_t at)
{
    const float z = p.f16 ? __half2float(static_cast<const __half *>(p.logits)[at]) : static_cast<const float *>(p.logits)[at];
    return z > -INFINITY ? z + 0.0f : -INFINITY;   // NaN -> masked; -0 -> +0
}

template <typename F> __device__ __forceinline__ F warp_max(F v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const F w = __shfl_xor_sync(kFull, v, o);
        v = w > v ? w : v;
    }
    return v;
}

// The token's chosen experts: lane s < k gets the expert of slot s. Returns whether
// the choice holds for the exact values (always for F = double).
template <typename F, int PER>
__device__ __forceinline__ bool choose(const Params &p, const float (&z)[PER], uint32_t lane, F *sv, uint32_t &mine)
{
    const F inf = Num<F>::inf();
    F v[PER];
    if (p.by_logit) {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = (F)z[j];
    } else {
        if (p.sigmoid) {
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = Num<F>::rcp((F)1 + Num<F>::exp(-(F)z[j]));
        } else {
            float zm = z[0];
#pragma unroll
            for (int j = 1; j < PER; ++j) zm = fmaxf(zm, z[j]);
            zm = warp_max(zm);
            F sum = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                v[j] = z[j] == zm ? (F)1 : Num<F>::exp((F)z[j] - (F)zm);
                if (z[j] == -INFINITY) v[j] = 0;
                sum += v[j];
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
            const F r = sum > (F)0 ? (F)1 / sum : (F)0;
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] *= r;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t e = lane + 32 * j;
            if (p.bias && e < p.E) v[j] += (F)p.bias[e];
            if (!(z[j] > -INFINITY) || !(v[j] == v[j])) v[j] = -inf;
            v[j] += (F)0;
        }
    }
    bool sure = true;
    const bool check = sizeof(F) == 4 && !p.by_logit;
    uint32_t keep = kFull;   // groups that stay
    if (p.top_groups < p.groups) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (lane + 32 * j < p.E) sv[lane + 32 * j] = v[j];
        __syncwarp();
        // lane g: the two largest of group g (groups <= 32)
        F b0 = -inf, b1 = -inf;
        if (lane < p.groups) {
            const F *s = sv + lane * p.group_size;
            uint32_t at = lane % p.group_size;   // start apart: groups of a power of two share a bank
            for (uint32_t i = 0; i < p.group_size; ++i) {
                const F x = s[at];
                at = at + 1 == p.group_size ? 0 : at + 1;
                b1 = x > b0 ? b0 : (x > b1 ? x : b1);
                b0 = x > b0 ? x : b0;
            }
        }
        __syncwarp();
        const F worth = p.group_top == 2 && p.group_size > 1 ? b0 + b1 : b0;
        uint32_t rank = 0;
        F edge = inf;   // distance to the nearest group on the other side of the cut
        for (uint32_t g = 0; g < p.groups; ++g) {
            const F w = __shfl_sync(kFull, worth, g);
            if (w > worth || (w == worth && g < lane)) ++rank;
        }
        const bool in = lane < p.groups && rank < p.top_groups;
        keep = __ballot_sync(kFull, in);
        if (check) {
            const uint32_t last = __ballot_sync(kFull, lane < p.groups && rank == p.top_groups - 1);
            const uint32_t next = __ballot_sync(kFull, lane < p.groups && rank == p.top_groups);
            const F a = __shfl_sync(kFull, worth, __ffs(last) - 1), b = __shfl_sync(kFull, worth, __ffs(next) - 1);
            edge = a - b;
            sure = edge > (F)(2 * kTol) * ((F)1 + (a < 0 ? -a : a));
        }
    }
    // repeated arg-max; taken and dropped experts leave through `open`
    uint32_t open = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t e = lane + 32 * j;
        if (e < p.E && (keep == kFull || keep >> (e / p.group_size) & 1u)) open |= 1u << j;
    }
    F before = inf;
    const uint32_t rounds = check ? p.k + 1 : p.k;
    for (uint32_t s = 0; s < rounds; ++s) {
        F bv = -inf;
        uint32_t be = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (open >> j & 1u && (v[j] > bv || be == 0xffffffffu)) {
                bv = v[j];
                be = lane + 32 * j;
            }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const F ov = __shfl_xor_sync(kFull, bv, o);
            const uint32_t oe = __shfl_xor_sync(kFull, be, o);
            if (oe != 0xffffffffu && (be == 0xffffffffu || ov > bv || (ov == bv && oe < be))) {
                bv = ov;
                be = oe;
            }
        }
        if (be == 0xffffffffu) break;   // only the extra round can run out of experts
        if (check && s) sure = sure && (before - bv > (F)(2 * kTol) * ((F)1 + (bv < 0 ? -bv : bv)));
        before = bv;
        if (s < p.k) {
            if (lane == s) mine = be;
            if (be % 32 == lane) open &= ~(1u << (be / 32));
        }
    }
    return sure;
}

template <int PER>
__global__ void __launch_bounds__(32 * kWarps) gate_kernel(const Params p)
{
    extern __shared__ double smem[];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double *sv = smem + (size_t)warp * p.E;
    const uint32_t t = blockIdx.x * kWarps + warp;
    if (t >= p.T) return;
    const size_t row = (size_t)t * p.E;
    float z[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) z[j] = lane + 32 * j < p.E ? load_logit(p, row + lane + 32 * j) : -INFINITY;
    uint32_t e = 0;
    if (!choose<float, PER>(p, z, lane, reinterpret_cast<float *>(sv), e)) choose<double, PER>(p, z, lane, sv, e);

    // weights of the chosen: lane s has slot s
    const bool have = lane < p.k;
    float zc = have ? load_logit(p, row + e) : -INFINITY, w = 0.0f, sum;
    if (p.renorm) {
        // relative to the largest chosen logit, so that scores too small for fp32 keep their ratio
        const float m = warp_max(zc);
        const bool low = !p.sigmoid || m < 0.0f;
        if (zc > -INFINITY) {
            w = low ? (zc == m ? 1.0f : expf(zc - m)) : 1.0f;
            if (p.sigmoid) w = __fdiv_rn(w, 1.0f + (low ? expf(zc) : expf(-zc)));
        }
        sum = w;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    } else if (p.sigmoid) {
        w = __fdiv_rn(1.0f, 1.0f + expf(-zc));
        sum = 1.0f;
    } else {
        float m = z[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) m = fmaxf(m, z[j]);
        m = warp_max(m);
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += z[j] > -INFINITY ? (z[j] == m ? 1.0f : expf(z[j] - m)) : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        if (zc > -INFINITY) w = zc == m ? 1.0f : expf(zc - m);
    }
    if (have) {
        p.ids[(size_t)t * p.k + lane] = (int32_t)e;
        p.weights[(size_t)t * p.k + lane] = sum > 0.0f ? __fdiv_rn(w, sum) * p.scale : 0.0f;
    }
}

}  // namespace gate

cudaError_t launch_moe_gate(const GateLaunch &L, cudaStream_t st)
{
    using namespace gate;
    if (!L.T) return cudaSuccess;
    Params p;
    p.logits = L.logits; p.bias = L.bias; p.ids = L.ids; p.weights = L.weights;
    p.T = L.T; p.E = L.E; p.k = L.k;
    p.groups = L.groups; p.top_groups = L.top_groups; p.group_top = L.group_top; p.group_size = L.E / L.groups;
    p.sigmoid = L.sigmoid; p.renorm = L.renorm; p.f16 = L.f16;
    // one score's order is its logit's; only a bias or a sum of two needs the scores
    p.by_logit = !L.bias && (L.top_groups == L.groups || L.group_top == 1 || p.group_size == 1);
    p.scale = L.scale;
    const unsigned grid = (L.T + kWarps - 1) / kWarps;
    const size_t smem = L.top_groups < L.groups ? (size_t)kWarps * L.E * sizeof(double) : 0;
    if (L.E <= 64) gate_kernel<2><<<grid, 32 * kWarps, smem, st>>>(p);
    else if (L.E <= 128) gate_kernel<4><<<grid, 32 * kWarps, smem, st>>>(p);
    else if (L.E <= 256) gate_kernel<8><<<grid, 32 * kWarps, smem, st>>>(p);
    else gate_kernel<16><<<grid, 32 * kWarps, smem, st>>>(p);
    return cudaGetLastError();
}

}  // namespace mpp41
