// Expert routing: scores (softmax or sigmoid), a balance bias that only the
// selection sees, expert groups, top-k and renormalised weights, one warp a token.
//
// Selection value of expert e: v = score + bias (-inf where the logit is -inf or
// NaN: a masked expert). With groups, a group's worth is the sum of its group_top
// largest v; the top_groups best groups stay, and the top_k experts are taken
// from them by falling v, ties to the lower index.
//
// The selection is exact: it is the one the 64-bit values give. Without a bias v is
// monotone in the logit, so experts (and groups by their best expert) are compared by
// the logits themselves. Otherwise fp32 scores decide, and wherever two values that
// the outcome depends on lie closer than the fp32 error, that warp decides the
// token again in 64 bits (exact_token, 2 to 3 us): about one token in a thousand for
// scores of a trained router's spread.
//
// fast_kernel: a lane holds PER neighbouring experts (16-byte loads), sorted once by
// 32-bit keys that carry the position in their lowest bits; each of the k rounds is
// then one warp-wide maximum of the lanes' heads and a shift in the winner's lane.
// A group is a run of lanes, its two best a butterfly; groups that do not fall on lane
// borders go through shared memory. 32768 tokens of 256 experts (8 of 4 of 8 groups) take
// 43.5 us, bound by the SMs and not by the 34 MB they read: 796 instructions a token are
// 22.5 us of issue slots, of which 66 % are used while an SM is active (waiting on the step
// before and on loads); the mean SM is active for three quarters of the time, the slowest
// for nine tenths. Logits without near ties take as long, the next token's logits loaded
// ahead changed nothing. A thread a token took 91 us.
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
    int sigmoid, renorm, f16;
    int by_logit;                         // experts are compared by their logits (no bias)
    int scores;                           // scores are needed: a bias, or sums of two for the groups
    int vec;                              // rows of logits start on 16 bytes
    float scale;
};

// Hardware exponential and reciprocal (2 ulp and 1 ulp), results below 2^-126 as 0.
__device__ __forceinline__ float fast_exp(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}

__device__ __forceinline__ float fast_rcp(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

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

// Order-preserving bits of a double (not NaN); never 0.
__device__ __forceinline__ unsigned long long order_bits64(double v)
{
    const long long u = __double_as_longlong(v);
    return (unsigned long long)(u ^ ((u >> 63) | (long long)0x8000000000000000ull));
}

// One token decided in 64 bits, experts lane + 32 j, j < PER. sv: E doubles of shared
// memory where groups are dropped. Lane s < k returns the expert of slot s. Built for
// latency: a token that comes here holds up its warp's others.
template <int PER>
__device__ __noinline__ uint32_t exact_token(const Params &p, size_t row, uint32_t lane, double *sv)
{
    const double inf = (double)INFINITY;
    double v[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = lane + 32 * j < p.E ? (double)load_logit(p, row + lane + 32 * j) : -inf;
    if (p.scores) {
        uint32_t masked = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) masked |= v[j] > -inf ? 0u : 1u << j;
        if (p.sigmoid) {
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = 1.0 / (1.0 + exp(-v[j]));
        } else {
            double m = v[0], sum = 0.0;
#pragma unroll
            for (int j = 1; j < PER; ++j) m = fmax(m, v[j]);
            m = warp_max(m);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                v[j] = masked >> j & 1u ? 0.0 : (v[j] == m ? 1.0 : exp(v[j] - m));
                sum += v[j];
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
            sum = sum > 0.0 ? sum : 1.0;
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] /= sum;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (p.bias && lane + 32 * j < p.E) v[j] += (double)p.bias[lane + 32 * j];
            if (masked >> j & 1u || !(v[j] == v[j])) v[j] = -inf;
        }
    }
    uint32_t keep = kFull;   // groups that stay
    if (p.top_groups < p.groups) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (lane + 32 * j < p.E) sv[lane + 32 * j] = v[j];
        __syncwarp();
        // the two largest of each group: `lanes` lanes a group (a power of two), each
        // taking every lanes-th of its experts
        uint32_t lanes = 32;
        while (lanes * p.groups > 32 && lanes > 1) lanes >>= 1;
        const uint32_t g = lane / lanes, sub = lane % lanes;
        double b0 = -inf, b1 = -inf;
        if (g < p.groups)
            for (uint32_t i = sub; i < p.group_size; i += lanes) {
                const double x = sv[g * p.group_size + i];
                b1 = fmax(b1, fmin(b0, x));
                b0 = fmax(b0, x);
            }
        for (uint32_t o = lanes >> 1; o; o >>= 1) {
            const double o0 = __shfl_xor_sync(kFull, b0, o), o1 = __shfl_xor_sync(kFull, b1, o);
            b1 = fmax(fmin(b0, o0), fmax(b1, o1));
            b0 = fmax(b0, o0);
        }
        double worth = p.group_top == 2 && p.group_size > 1 ? b0 + b1 : b0;
        if (!(worth > -inf)) worth = -inf;   // inf - inf
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < p.groups; ++i) {
            const double w = __shfl_sync(kFull, worth, i * lanes);
            rank += w > worth || (w == worth && i < g) ? 1u : 0u;
        }
        const uint32_t in = __ballot_sync(kFull, g < p.groups && rank < p.top_groups);
        keep = 0u;   // bit g from its first lane
        for (uint32_t i = 0; i < p.groups; ++i) keep |= (in >> (i * lanes) & 1u) << i;
        __syncwarp();
    }
    // repeated arg-max by 64-bit keys: upper half, lower half, then the lowest expert; 0 = not open
    unsigned long long key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t e = lane + 32 * j;
        if (p.by_logit && p.scores && e < p.E) v[j] = (double)load_logit(p, row + e);
        key[j] = e < p.E && (keep == kFull || keep >> (e / p.group_size) & 1u) ? order_bits64(v[j] + 0.0) : 0ull;
    }
    uint32_t mine = 0;
    for (uint32_t s = 0; s < p.k; ++s) {
        unsigned long long h = key[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) h = key[j] > h ? key[j] : h;
        const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(h >> 32));
        const uint32_t lo = __reduce_max_sync(kFull, (uint32_t)(h >> 32) == hi ? (uint32_t)h : 0u);
        const unsigned long long m = (unsigned long long)hi << 32 | lo;
        uint32_t e = kFull;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) e = key[j] == m ? lane + 32 * j : e;
        e = __reduce_min_sync(kFull, e);
        if (lane == s) mine = e;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (lane + 32 * j == e) key[j] = 0ull;
    }
    __syncwarp();
    return mine;
}

// Weight of the lane's chosen expert e: lanes come in runs of kp (a power of two, at least
// k), one run a token t, the lane's slot in it s. zmax and zsum: softmax's maximum and
// sum over all experts, used without renormalisation. live: the run has a token.
__device__ __forceinline__ void write_slot(const Params &p, size_t t, uint32_t s, uint32_t kp, bool live, uint32_t e, float zmax,
                                           float zsum)
{
    const bool have = live && s < p.k;
    const float zc = have ? load_logit(p, t * p.E + e) : -INFINITY;
    float w = 0.0f, sum;
    if (p.renorm) {
        // relative to the largest chosen logit, so that scores too small for fp32 keep their ratio
        float m = zc;
        for (uint32_t o = kp >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        const bool low = !p.sigmoid || m < 0.0f;
        if (zc > -INFINITY) {
            w = low ? (zc == m ? 1.0f : expf(zc - m)) : 1.0f;
            if (p.sigmoid) w = __fdiv_rn(w, 1.0f + (low ? expf(zc) : expf(-zc)));
        }
        sum = w;
        for (uint32_t o = kp >> 1; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    } else if (p.sigmoid) {
        w = __fdiv_rn(1.0f, 1.0f + expf(-zc));
        sum = 1.0f;
    } else {
        if (zc > -INFINITY) w = zc == zmax ? 1.0f : expf(zc - zmax);
        sum = zsum;
    }
    if (have) {
        p.ids[t * p.k + s] = (int32_t)e;
        p.weights[t * p.k + s] = sum > 0.0f ? __fdiv_rn(w, sum) * p.scale : 0.0f;
    }
}

// Softmax's maximum and sum (accurate exponentials) over the lanes' z.
template <int PER> __device__ __forceinline__ void softmax_norm(const float (&z)[PER], float &m, float &sum)
{
    m = z[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) m = fmaxf(m, z[j]);
    m = warp_max(m);
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += z[j] > -INFINITY ? (z[j] == m ? 1.0f : expf(z[j] - m)) : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
}

// Order-preserving bits of a float (not NaN); never 0.
__device__ __forceinline__ uint32_t order_bits(float v)
{
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float order_value(uint32_t k)
{
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__host__ __device__ constexpr int key_bits(int per) { return per <= 1 ? 0 : per <= 2 ? 1 : per <= 4 ? 2 : per <= 8 ? 3 : 4; }

// Batcher's odd-even merge sort, descending, of any N (comparators beyond N are left out).
template <int N> __device__ __forceinline__ void sort_desc(uint32_t (&k)[N])
{
#pragma unroll
    for (int p = 1; p < N; p <<= 1)
#pragma unroll
        for (int q = p; q >= 1; q >>= 1)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t a = k[i + j], b = k[i + j + q];
                        k[i + j] = max(a, b);
                        k[i + j + q] = min(a, b);
                    }
}

template <int PER, bool F16>
__device__ __forceinline__ void load_lane(const Params &p, uint32_t t, uint32_t lane, float (&z)[PER])
{
    const size_t at = (size_t)t * p.E + lane * PER;
    if (PER % 4 == 0 && p.vec && p.E % PER == 0) {   // whole lanes, on 8 bytes at least
        const bool have = lane * PER < p.E;
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) {
            float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (have) {
                if (F16) {
                    const uint2 h = __ldg(reinterpret_cast<const uint2 *>(static_cast<const __half *>(p.logits) + at) + j);
                    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h.x));
                    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
                    v = make_float4(a.x, a.y, b.x, b.y);
                } else {
                    v = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p.logits) + at) + j);
                }
            }
            z[4 * j] = v.x; z[4 * j + 1] = v.y; z[4 * j + 2] = v.z; z[4 * j + 3] = v.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        z[j] = -INFINITY;
        if (lane * PER + j < p.E)
            z[j] = F16 ? __half2float(static_cast<const __half *>(p.logits)[at + j]) : static_cast<const float *>(p.logits)[at + j];
    }
}

// lanes: where groups are dropped, the lanes a group takes (a power of two): its experts
// lie in them, or (SMEM_GROUPS) they read them from shared memory; else 0.
// A warp chooses for `batch` tokens, one after the other, and then weighs their choices
// together, kp lanes a token (batch * kp <= 32).
template <int PER, bool F16, bool SMEM_GROUPS>
__global__ void __launch_bounds__(32 * kWarps, PER <= 8 ? 7 : 5) fast_kernel(const Params p, uint32_t lanes, uint32_t batch, uint32_t kp)
{
    extern __shared__ double smem[];
    __shared__ uint32_t sel[kWarps][32];
    __shared__ float2 norm[kWarps][32];
    constexpr int kBits = key_bits(PER);
    constexpr uint32_t kLow = (1u << kBits) - 1u;
    constexpr int kExactPer = PER <= 2 ? 2 : PER <= 4 ? 4 : PER <= 8 ? 8 : 16;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double *sv = smem + (size_t)warp * p.E;
    const uint32_t stride = gridDim.x * kWarps * batch;
    pdl_wait_prior();
    float bias[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        bias[j] = p.bias && lane * PER + j < p.E ? p.bias[lane * PER + j] : 0.0f;
        if (!(bias[j] > -INFINITY)) bias[j] = -INFINITY;   // NaN: as a masked expert
    }
    // How far two fp32 values have to be apart for their order to be the exact values'.
    // A score: ex2 (2^-22 of its value, and |x| 2^-24 by its argument) times the sigmoid's
    // slope or the softmax value stays below 2^-24 * 1.3, the sum 1 + e, the reciprocal and
    // the bias add half, one and half an ulp: below 2^-22 for values up to 2, both together
    // 2^-21 (and 2^-23 |v| for larger ones). A softmax's sum is off by one factor for all,
    // at most PER + 10 half ulps. Logits compared themselves have no error. Keys cut to
    // their upper bits keep the order; equal ones are less than one cut unit apart.
    const float err = (p.sigmoid ? 0.0f : (float)(PER + 10) / 16777216.0f) + 1.0f / 2097152.0f, tol = p.by_logit ? 0.0f : err;
    const float unit = ((float)(1u << kBits) + (p.by_logit ? 0.0f : 1.0f)) / 8388608.0f;
    const bool ragged = p.E % PER != 0 || lane * PER >= p.E;
    const float inv_size = __fdividef(1.0f, (float)p.group_size);
    const bool check = !(p.by_logit && F16);   // fp16 logits lose no bits to the position
    for (uint64_t t0 = (uint64_t)(blockIdx.x * kWarps + warp) * batch; t0 < p.T; t0 += stride) {
        const uint32_t n = (uint32_t)min((uint64_t)batch, p.T - t0);
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t t = (uint32_t)t0 + i;
            float z[PER], v[PER];
            load_lane<PER, F16>(p, t, lane, z);
            if (!p.scores) {
#pragma unroll
                for (int j = 0; j < PER; ++j) v[j] = z[j] > -INFINITY ? z[j] + 0.0f : -INFINITY;   // NaN masks; -0 -> +0
            } else if (p.sigmoid) {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    v[j] = fast_rcp(1.0f + fast_exp(-z[j])) + bias[j];
                    if (!(z[j] > -INFINITY)) v[j] = -INFINITY;
                }
            } else {
                float m = z[0];
#pragma unroll
                for (int j = 1; j < PER; ++j) m = fmaxf(m, z[j]);   // NaN is no maximum
                m = warp_max(m > -INFINITY ? m : -INFINITY);
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    v[j] = z[j] == m ? 1.0f : fast_exp(z[j] - m);
                    if (!(z[j] > -INFINITY)) v[j] = 0.0f;
                    sum += v[j];
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
                const float r = sum > 0.0f ? fast_rcp(sum) : 0.0f;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    v[j] = v[j] * r + bias[j];
                    if (!(z[j] > -INFINITY)) v[j] = -INFINITY;
                }
            }
            bool sure = true;
            uint32_t stay = kFull;   // bit g: group g stays
            if (lanes) {
                float b0 = -INFINITY, b1 = -INFINITY;
                const uint32_t mine = lane / lanes;
                if constexpr (!SMEM_GROUPS) {
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        b1 = fmaxf(b1, fminf(b0, v[j]));
                        b0 = fmaxf(b0, v[j]);
                    }
                } else {
                    float *sf = reinterpret_cast<float *>(sv);
#pragma unroll
                    for (int j = 0; j < PER; ++j)
                        if (lane * PER + j < p.E) sf[lane * PER + j] = v[j];
                    __syncwarp();
                    if (mine < p.groups)
                        for (uint32_t q = lane % lanes; q < p.group_size; q += lanes) {
                            const float x = sf[mine * p.group_size + q];
                            b1 = fmaxf(b1, fminf(b0, x));
                            b0 = fmaxf(b0, x);
                        }
                    __syncwarp();
                }
                for (uint32_t o = lanes >> 1; o; o >>= 1) {
                    const float o0 = __shfl_xor_sync(kFull, b0, o), o1 = __shfl_xor_sync(kFull, b1, o);
                    b1 = fmaxf(fminf(b0, o0), fmaxf(b1, o1));
                    b0 = fmaxf(b0, o0);
                }
                const bool two = p.group_top == 2 && p.group_size > 1;
                float worth = two ? b0 + b1 : b0;
                if (!(worth > -INFINITY)) worth = -INFINITY;   // inf - inf
                uint32_t rank = 0;
                if (!p.scores) {
                    for (uint32_t g = 0; g < p.groups; ++g) {
                        const float w = __shfl_sync(kFull, worth, g * lanes);
                        rank += w > worth || (w == worth && g < mine) ? 1u : 0u;
                    }
                } else {   // groups tied at the cut all stay: too many, which is not sure
#pragma unroll 4
                    for (uint32_t g = 0; g < p.groups; ++g)
                        rank += __shfl_sync(kFull, worth, g * lanes) > worth ? 1u : 0u;
                }
                const bool real = mine < p.groups;
                const bool keep = real && rank < p.top_groups;
                const uint32_t in_lanes = __ballot_sync(kFull, keep);
                if constexpr (!SMEM_GROUPS) {
                    stay = keep ? kFull : 0u;   // of this lane's group
                } else {
                    stay = 0u;
                    for (uint32_t g = 0; g < p.groups; ++g) stay |= (in_lanes >> (g * lanes) & 1u) << g;
                }
                if (p.scores) {
                    // The last group that stays and the first that goes have to be well apart.
                    // A worth is off by its scores' errors (err covers two) and by half an ulp of
                    // each addend and of the sum, whose own size says nothing of theirs where
                    // they have opposite signs: 2^-23 of both addends' sizes, here 2^-22.
                    const float far = err + (fabsf(b0) + (two ? fabsf(b1) : 0.0f)) * (1.0f / 4194304.0f);
                    const float off = fabsf(worth) < INFINITY ? far : 0.0f;   // infinite worths are exact
                    const float in = order_value(__reduce_min_sync(kFull, keep ? order_bits(worth - off) : 0xFFFFFFFFu));
                    const float out = order_value(__reduce_max_sync(kFull, real && !keep ? order_bits(worth + off) : 0u));
                    sure = __popc(in_lanes) == p.top_groups * lanes && in > out;
                }
            }
            uint32_t key[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                float x = v[j];
                if (p.by_logit && p.scores) x = z[j] > -INFINITY ? z[j] + 0.0f : -INFINITY;
                key[j] = (order_bits(x) & ~kLow) | (kLow - (uint32_t)j);
                if constexpr (SMEM_GROUPS) {
                    // e / group_size by the reciprocal: exact below 512
                    const uint32_t g = (uint32_t)(((float)(lane * PER + j) + 0.5f) * inv_size);
                    if (!(stay >> (g & 31u) & 1u)) key[j] = 0u;
                } else if (!stay) {
                    key[j] = 0u;
                }
                if (ragged && lane * PER + j >= p.E) key[j] = 0u;
            }
            sort_desc<PER>(key);
            uint32_t won = 0, pops = 0;   // lane s: the winning key of round s; heads this lane gave
            uint32_t *out = &sel[warp][i * kp];
            for (uint32_t s = 0; s < p.k; ++s) {
                const uint32_t m = __reduce_max_sync(kFull, key[0]);
                bool win = key[0] == m;
                if (!check) {
                    // ties are exact here: the lowest lane has the lowest expert
                    const uint32_t first = __ffs(__ballot_sync(kFull, (key[0] >> kBits) == (m >> kBits))) - 1;
                    win = lane == first;
                }
                if (lane == s) won = m;
                if (win) {
                    out[s] = lane * PER + (kLow - (key[0] & kLow));
                    ++pops;
                }
#pragma unroll
                for (int j = 0; j + 1 < PER; ++j) key[j] = win ? key[j + 1] : key[j];
                if (win) key[PER - 1] = 0u;
            }
            if (check) {
                // neighbours in the order, the first not chosen among them, have to be apart
                const uint32_t after = __reduce_max_sync(kFull, key[0]);
                uint32_t next = __shfl_down_sync(kFull, won, 1);
                sure = sure && __reduce_add_sync(kFull, pops) == p.k;   // two lanes with one key
                if (lane + 1 == p.k) next = after;
                if (lane < p.k && next != 0u) {
                    const float a = order_value(won & ~kLow), b = order_value(next & ~kLow);
                    sure = sure && (won >> kBits) != (next >> kBits) && a - b > tol + fmaxf(fabsf(a), fabsf(b)) * unit * (p.by_logit ? 0.0f : 1.0f);
                }
            }
            if (check || p.scores) {
                if (!__all_sync(kFull, sure)) {
                    __syncwarp();
                    const uint32_t e = exact_token<kExactPer>(p, (size_t)t * p.E, lane, sv);
                    if (lane < p.k) sel[warp][i * kp + lane] = e;
                }
            }
            if (!p.renorm && !p.sigmoid) {
                float m, sum;
#pragma unroll
                for (int j = 0; j < PER; ++j) z[j] = z[j] > -INFINITY ? z[j] : -INFINITY;
                softmax_norm<PER>(z, m, sum);
                if (lane == 0) norm[warp][i] = make_float2(m, sum);
            }
        }
        __syncwarp();
        const uint32_t i = lane / kp, s = lane % kp;
        const bool live = i < n;
        const float2 nm = live ? norm[warp][i] : make_float2(0.0f, 1.0f);
        write_slot(p, t0 + i, s, kp, live, live && s < p.k ? sel[warp][i * kp + s] : 0u, nm.x, nm.y);
        __syncwarp();
    }
}

template <bool F16, bool SMEM_GROUPS> cudaError_t launch_fast(const Params &p, uint32_t per, uint32_t lanes, cudaStream_t st)
{
    // Weighing a token's k choices leaves most lanes idle: from enough tokens for every
    // warp slot, a warp weighs as many together as fit its lanes.
    uint32_t kp = 1;
    while (kp < p.k) kp *= 2;
    const uint32_t most = 148 * 7, batch = p.T >= most * kWarps ? 32 / kp : 1;
    const uint64_t per_cta = (uint64_t)kWarps * batch, want = (p.T + per_cta - 1) / per_cta;
    const unsigned grid = (unsigned)(want < most ? want : most);
    const size_t smem = lanes ? (size_t)kWarps * p.E * sizeof(double) : 0;
    switch (per) {
#define GATE_CASE(N) case N: return launch_overlapped(fast_kernel<N, F16, SMEM_GROUPS>, dim3(grid), dim3(32 * kWarps), smem, st, p, lanes, batch, kp);
    GATE_CASE(1) GATE_CASE(2) GATE_CASE(3) GATE_CASE(4) GATE_CASE(5) GATE_CASE(6) GATE_CASE(8) GATE_CASE(10) GATE_CASE(12)
    GATE_CASE(16)
#undef GATE_CASE
    }
    return cudaErrorInvalidValue;
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
    p.by_logit = !L.bias;
    p.scores = L.bias || (L.top_groups < L.groups && L.group_top == 2 && p.group_size > 1);
    p.scale = L.scale;
    p.vec = (size_t)L.E * (L.f16 ? 2 : 4) % 16 == 0 && (reinterpret_cast<uintptr_t>(L.logits) & 15u) == 0;
    const bool grouped = L.top_groups < L.groups;
    // Experts a lane: the fewest that hold all; where groups are dropped rather up to twice
    // that, if a group then lies in a power of two of lanes.
    uint32_t per = 0, lanes = 0, least = 0;
    for (uint32_t c : {1u, 2u, 3u, 4u, 5u, 6u, 8u, 10u, 12u, 16u}) {
        if (c * 32 < L.E) continue;
        if (!least) least = c;
        const uint32_t in = p.group_size / c;
        if (!grouped || (c <= 2 * least && p.group_size % c == 0 && !(in & (in - 1)))) {
            per = c;
            lanes = grouped ? in : 0;
            break;
        }
    }
    if (per) return L.f16 ? launch_fast<true, false>(p, per, lanes, st) : launch_fast<false, false>(p, per, lanes, st);
    lanes = 32;
    while (lanes * p.groups > 32 && lanes > 1) lanes >>= 1;
    return L.f16 ? launch_fast<true, true>(p, least, lanes, st) : launch_fast<false, true>(p, least, lanes, st);
}

}  // namespace mpp41
