// FP8 matrix product with a scale per block of 128 along K:
//   C[m][n] = sum_kb sa[m][kb] * sb[n / 128][kb] * sum_{k in block kb} A[m][k] * B[n][k]
// A [M][K] and B [N][K] are E4M3 or E5M2 (each its own), sa [M][K/128] fp32 (one
// scale per row and block), sb [N/128][K/128] fp32 (one per 128 x 128 block). The
// scales are arbitrary fp32 numbers, so they cannot ride in the MMA's E8M0 block
// scales: the tensor core sums one 128-wide K block into a fresh fp32 accumulator
// in tensor memory (tcgen05.mma kind::f8f6f4, four K = 32 steps), and eight
// promotion warps read it back, multiply it by sa * sb and add it to fp32
// registers while the MMAs of the next block fill the other accumulator.
//
// Grouped form: rows [offsets[g], offsets[g+1]) of A meet B[g]; every CTA builds
// the prefix sums of the groups' row tiles in shared memory, so the tile walk
// needs no host knowledge of the offsets and no second launch.
//
// Tile: 128 rows (MMA M) x BN columns (MMA N). Rows are the M side for every row
// count: a thread then owns one row, and the promotion's scale is one register
// pair instead of a shared-memory read per column. Row blocks past the tile's end
// are neither loaded nor promoted (32-row granularity).
//
// Warp roles (384 threads): 0 TMA producer, 1 MMA issuer and TMEM owner, 2..3
// idle, 4..11 promotion (warp w: TMEM lane quarter w % 4, column half (w - 4) / 4).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "mpp41_device.cuh"
#include "mpp41_fp8.cuh"
#include "mpp41_internal.h"

namespace mpp41 {
namespace fp8 {

constexpr uint32_t kBM = 128;
constexpr uint32_t kBK = 128;               // one scale block, one 128-byte swizzle atom
constexpr int kThreads = 384;
constexpr int kPromoThreads = 256;
constexpr uint32_t kBoxRows = 32;           // rows of A per TMA box
constexpr uint32_t kBoxBytes = kBoxRows * kBK;
constexpr uint32_t kBTile = 128 * kBK;      // 128 rows of B

enum Epi { EPI_STORE = 0, EPI_SWIGLU = 1 };

// AR: rows of A a stage has room for. With AR = 32 (at most 32 rows in the whole
// launch) the MMA still reads 128 rows from the stage's start: the other 96 come
// from the neighbouring stages and only reach accumulator lanes nobody reads.
template <int BN, int AR> struct Cfg {
    static constexpr uint32_t kAStage = AR * kBK;
    static constexpr uint32_t kBStage = BN * kBK;
    static constexpr int kStages = BN == 256 ? 4 : (AR == 32 ? 9 : 6);
    static constexpr uint32_t kOffB = ((kStages * kAStage + 1023) / 1024) * 1024;
    static constexpr uint32_t kOffBar = kOffB + kStages * kBStage;
    static constexpr uint32_t kOffAmax = kOffBar + 256;             // SwiGLU: [2 tiles][2 halves][128] floats
    static constexpr uint32_t kOffGroups = kOffAmax + 2048;         // 3 words per group + 1
    static constexpr uint32_t kSmem = 1024 + kOffGroups;            // + 4 * (3 * groups + 1)
    static constexpr uint32_t kTmemCols = 2 * BN;
    static_assert(AR * kBK * (kStages - 1) + 128 * kBK <= kOffB + kStages * kBStage, "MMA reads stay inside the ring");
    static_assert(kSmem <= 227 * 1024 - 4 * (3 * 1024 + 1), "shared memory");
};

struct Params {
    CUtensorMap tm_a;           // A [M][K], box {128, 32}, SW128
    CUtensorMap tm_b0, tm_b1;   // B [groups * N][K], box {128, 128}, SW128 (tm_b1: the up weights, SwiGLU)
    const float *sa;            // [M][kb]
    const float *sb0, *sb1;     // [groups][nb][kb]
    const int32_t *offsets;     // [groups + 1] or null (one group of M rows)
    void *out;                  // C [M][N], or the 8-bit mid [M][N] of the SwiGLU form
    float *out_scales;          // SwiGLU: [M][nb]
    uint32_t M, N, K, kb, nb, groups, n_tiles;
    uint32_t idesc;
    int out_f16;
    int out_fmt;                // SwiGLU: 8-bit format of the mid (FMT_*)
    int vec;                    // rows of C start on 16-byte boundaries
    uint32_t *err;
};

// Instruction descriptor, kind::f8f6f4, fp32 D, both operands K-major; formats 0 = E4M3, 1 = E5M2.
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N, uint32_t af, uint32_t bf)
{
    return (1u << 4) | (af << 7) | (bf << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Completion of this thread's tcgen05.ld, tied to the registers it fills so that no use moves above it.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// acc[i] += d[2i..2i+1] * s for 16 fp32 pairs (packed fp32 FMA: two per instruction).
__device__ __forceinline__ void promote32(uint64_t *acc, const uint32_t (&d)[32], uint64_t s2)
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        uint64_t v;
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(d[2 * i]), "r"(d[2 * i + 1]));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i]) : "l"(v), "l"(s2));
    }
}

__device__ __forceinline__ uint64_t pack2(float s)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %1};" : "=l"(v) : "f"(s));
    return v;
}

__device__ __forceinline__ float2 unpack2(uint64_t v)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}

// Barrier of the promotion warps that also ORs a flag.
__device__ __forceinline__ bool promo_any(bool v)
{
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)v), "n"(kPromoThreads) : "memory");
    return r != 0;
}

// ---- the tile walk
struct Groups {
    const uint32_t *cum;    // [groups + 1] row tiles before group g
    const uint32_t *row0;   // [groups]
    const uint32_t *row1;   // [groups]
};

struct Tile {
    uint32_t g, m0, m_end, n0;
};

// Tile t: groups in order; inside a group the row tile runs fastest, so that the
// CTAs of a wave share the weight tile they stream.
__device__ __forceinline__ Tile tile_at(const Params &p, const Groups &gr, uint32_t t, uint32_t cols)
{
    uint32_t lo = 0, hi = p.groups;   // cum[lo] * n_tiles <= t < cum[hi] * n_tiles
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (gr.cum[mid] * p.n_tiles <= t) lo = mid; else hi = mid;
    }
    const uint32_t mt = gr.cum[lo + 1] - gr.cum[lo];
    const uint32_t l = t - gr.cum[lo] * p.n_tiles;
    Tile o;
    o.g = lo;
    o.m0 = gr.row0[lo] + (l % mt) * kBM;
    o.m_end = gr.row1[lo];
    o.n0 = (l / mt) * cols;
    return o;
}

// Prefix sums of the groups' row tiles (one warp). Offsets are clamped to [0, M]
// and made ascending, so wrong ones are reported but never lead out of A or C.
__device__ __forceinline__ void build_groups(const Params &p, uint32_t *cum, uint32_t *row0, uint32_t *row1, uint32_t lane)
{
    const uint32_t per = (p.groups + 31) / 32;
    uint32_t sum = 0;
    bool bad = false;
    for (uint32_t i = 0; i < per; ++i) {
        const uint32_t g = lane * per + i;
        if (g >= p.groups) break;
        uint32_t a = 0, b = p.M;
        if (p.offsets) {
            const int32_t o0 = p.offsets[g], o1 = p.offsets[g + 1];
            a = (uint32_t)min(max((int64_t)o0, (int64_t)0), (int64_t)p.M);
            b = (uint32_t)min(max((int64_t)o1, (int64_t)a), (int64_t)p.M);
            bad |= (int64_t)a != o0 || (int64_t)b != o1;
        }
        row0[g] = a;
        row1[g] = b;
        sum += (b - a + kBM - 1) / kBM;
    }
    if (bad && blockIdx.x == 0) report_error(p.err, kErrBounds, 0xF81);
    uint32_t inc = sum;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += v;
    }
    uint32_t base = inc - sum;
    for (uint32_t i = 0; i < per; ++i) {
        const uint32_t g = lane * per + i;
        if (g >= p.groups) break;
        cum[g] = base;
        base += (row1[g] - row0[g] + kBM - 1) / kBM;
    }
    if (lane == 31) cum[p.groups] = inc;
}

// A thread's run of 64 columns [c, c + 64) of row m.
__device__ __forceinline__ void store_run(const Params &p, const uint64_t *acc, uint32_t m, uint32_t c)
{
    const size_t at = (size_t)m * p.N + c;
    if (p.out_f16) {
        __half *o = static_cast<__half *>(p.out) + at;
        if (p.vec && c + 64 <= p.N) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 f = unpack2(acc[4 * i + q]);
                    w[q] = half2_bits(f.x, f.y);
                }
                reinterpret_cast<uint4 *>(o)[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float2 f = unpack2(acc[i]);
                if (c + 2 * i < p.N) o[2 * i] = __float2half_rn(f.x);
                if (c + 2 * i + 1 < p.N) o[2 * i + 1] = __float2half_rn(f.y);
            }
        }
    } else {
        float *o = static_cast<float *>(p.out) + at;
        if (p.vec && c + 64 <= p.N) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 f = unpack2(acc[2 * i]), h = unpack2(acc[2 * i + 1]);
                reinterpret_cast<float4 *>(o)[i] = make_float4(f.x, f.y, h.x, h.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float2 f = unpack2(acc[i]);
                if (c + 2 * i < p.N) o[2 * i] = f.x;
                if (c + 2 * i + 1 < p.N) o[2 * i + 1] = f.y;
            }
        }
    }
}

// SPLIT: one tile per cluster; the cluster's CTAs take equal ranges of K blocks
// and add their fp32 partials in rank order through distributed shared memory
// (few rows: the products of a weight stream alone would leave SMs idle).
template <int BN, int AR, int E, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Params p)
{
    using C = Cfg<BN, AR>;
    constexpr int S = C::kStages;
    constexpr uint32_t kRuns = BN / 128;     // 64-column runs per promotion thread
    constexpr uint32_t kCols = E == EPI_SWIGLU ? BN / 2 : BN;   // output columns per tile
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem, *sB = smem + C::kOffB;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kOffBar);
    uint64_t *full = bars, *empty = bars + S;
    uint64_t *acc_full = bars + 2 * S, *acc_empty = bars + 2 * S + 2, *drain = bars + 2 * S + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S + 5);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float *amax_x = reinterpret_cast<float *>(smem + C::kOffAmax);
    uint32_t *cum = reinterpret_cast<uint32_t *>(smem + C::kOffGroups);
    uint32_t *row0 = cum + p.groups + 1, *row1 = row0 + p.groups;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 8);
        }
        mbar_init(drain, 1);
        *abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_a);
        tma_prefetch_desc(&p.tm_b0);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    if (warp == 2) build_groups(p, cum, row0, row1, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Groups gr{cum, row0, row1};

    // SPLIT: blockIdx.x = tile * cluster + rank; K blocks [k0, k1) of this CTA
    uint32_t t0 = blockIdx.x, step = gridDim.x, k0 = 0, k1 = p.kb, rank = 0, parts = 1;
    if constexpr (SPLIT) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
        t0 = blockIdx.x / parts;
        step = gridDim.x / parts;
        k0 = (uint32_t)((uint64_t)p.kb * rank / parts);
        k1 = (uint32_t)((uint64_t)p.kb * (rank + 1) / parts);
    }
    const uint32_t total = cum[p.groups] * p.n_tiles;

    // BN = 256: 64 packed accumulators and 64 words in flight need more than the 168
    // registers a thread is launched with: 128 * 56 + 256 * 224 = 384 * 168
    if (warp < 4) {
        if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            // ------------------------------------------------ TMA producer
            uint32_t g = 0;
            bool alive = true;
            for (uint32_t t = t0; t < total && alive; t += step) {
                const Tile tl = tile_at(p, gr, t, kCols);
                const uint32_t rows = min(tl.m_end - tl.m0, kBM), boxes = (rows + kBoxRows - 1) / kBoxRows;
                const int32_t b_row = (int32_t)(tl.g * p.N + tl.n0);
                // the second 128 rows of B: the up weights, or the next columns (none behind the last)
                const bool second = BN == 256 && (E == EPI_SWIGLU || tl.n0 + 128 < p.N);
                const uint32_t bytes = boxes * kBoxBytes + (second ? 2 : 1) * kBTile;
                for (uint32_t kk = k0; kk < k1; ++kk, ++g) {
                    const uint32_t st = g % S, ph = (g / S) & 1u;
                    if (!warp_wait(&empty[st], ph ^ 1u, abort, p.err, 0xF01)) { alive = false; break; }
                    if (elect_one_sync()) {
                        mbar_arrive_expect_tx(&full[st], bytes);
                        const int32_t kc = (int32_t)(kk * kBK);
                        tma_load_2d(sB + st * C::kBStage, &p.tm_b0, kc, b_row, &full[st]);
                        if (second) {
                            if constexpr (E == EPI_SWIGLU)
                                tma_load_2d(sB + st * C::kBStage + kBTile, &p.tm_b1, kc, b_row, &full[st]);
                            else
                                tma_load_2d(sB + st * C::kBStage + kBTile, &p.tm_b0, kc, b_row + 128, &full[st]);
                        }
                        for (uint32_t i = 0; i < boxes; ++i)
                            tma_load_2d(sA + st * C::kAStage + i * kBoxBytes, &p.tm_a, kc,
                                        (int32_t)(tl.m0 + i * kBoxRows), &full[st]);
                    }
                    __syncwarp();
                }
            }
            // drain: no copy may still be landing when the CTA exits
            for (uint32_t q = (g > (uint32_t)S ? g - S : 0); q < g; ++q)
                mbar_wait(&full[q % S], (q / S) & 1u, nullptr, p.err, 0xF02);
        } else if (warp == 1) {
            // ------------------------------------------------ MMA issuer
            uint32_t g = 0;
            bool alive = true;
            for (uint32_t t = t0; t < total && alive; t += step) {
                for (uint32_t kk = k0; kk < k1; ++kk, ++g) {
                    const uint32_t st = g % S, ph = (g / S) & 1u, b = g & 1u;
                    if (!warp_wait(&acc_empty[b], ((g >> 1) & 1u) ^ 1u, abort, p.err, 0xF03) ||
                        !warp_wait(&full[st], ph, abort, p.err, 0xF04)) { alive = false; break; }
                    tc_fence_after();
                    if (elect_one_sync()) {
                        const uint64_t ad = smem_desc_sw128(sA + st * C::kAStage);
                        const uint64_t bd = smem_desc_sw128(sB + st * C::kBStage);
    #pragma unroll
                        for (uint32_t k = 0; k < kBK / 32; ++k)
                            mma_f8(tmem + b * BN, ad + 2 * k, bd + 2 * k, p.idesc, k != 0u);
                        mma_commit(&empty[st]);
                        mma_commit(&acc_full[b]);
                    }
                    __syncwarp();
                }
            }
            if (elect_one_sync()) mma_commit(drain);
            __syncwarp();
        }
    } else {
        if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ------------------------------------------------ promotion and epilogue
        const uint32_t quarter = warp & 3, half = (uint32_t)(warp - 4) >> 2;
        const uint32_t lane_base = (quarter * 32u) << 16;
        uint32_t g = 0, n_done = 0;
        bool alive = true;
        for (uint32_t t = t0; t < total && alive; t += step, ++n_done) {
            const Tile tl = tile_at(p, gr, t, kCols);
            const uint32_t m = tl.m0 + quarter * 32 + lane;
            const bool live = tl.m0 + quarter * 32 < tl.m_end;   // this warp's rows exist
            const bool row_ok = m < tl.m_end;
            // the thread's runs of 64 accumulator columns: run r starts at col(r)
            auto col = [&](uint32_t r) -> uint32_t { return E == EPI_SWIGLU ? r * 128 + half * 64 : half * (BN / 2) + r * 64; };
            const float *sa = p.sa + (size_t)(row_ok ? m : tl.m0) * p.kb;
            const float *sb[2];
            if constexpr (E == EPI_SWIGLU) {
                const size_t blk = ((size_t)tl.g * p.nb + tl.n0 / 128) * p.kb;
                sb[0] = p.sb0 + blk;
                sb[1] = p.sb1 + blk;
            } else {
                const uint32_t nblk = min((tl.n0 + col(0)) / 128, p.nb - 1);
                sb[0] = sb[1] = p.sb0 + ((size_t)tl.g * p.nb + nblk) * p.kb;
            }
            uint64_t acc[kRuns * 32];
#pragma unroll
            for (uint32_t i = 0; i < kRuns * 32; ++i) acc[i] = 0ull;
            // scales two blocks ahead: an L2 round trip is longer than one block's MMAs
            float a0 = 0.0f, a1 = 0.0f, u0 = 0.0f, u1 = 0.0f, w0 = 0.0f, w1 = 0.0f;
            auto fetch = [&](uint32_t kk, float &a, float &u, float &w) {
                if (live && kk < k1) {
                    a = __ldg(sa + kk);
                    u = __ldg(sb[0] + kk);
                    if constexpr (E == EPI_SWIGLU) w = __ldg(sb[1] + kk);
                }
            };
            fetch(k0, a0, u0, w0);
            fetch(k0 + 1, a1, u1, w1);
            for (uint32_t kk = k0; kk < k1; ++kk, ++g) {
                const uint32_t b = g & 1u;
                float a2 = 0.0f, u2 = 0.0f, w2 = 0.0f;
                fetch(kk + 2, a2, u2, w2);
                if (!warp_wait(&acc_full[b], (g >> 1) & 1u, abort, p.err, 0xF05)) { alive = false; break; }
                tc_fence_after();
                if (live) {
                    const uint32_t base = tmem + lane_base + b * BN;
                    const uint64_t s0 = pack2(a0 * u0), s1 = E == EPI_SWIGLU ? pack2(a0 * w0) : s0;
                    uint32_t d0[32], d1[32];
                    tmem_ld_32x32b_x32(base + col(0), d0);
                    tmem_ld_wait32(d0);
#pragma unroll
                    for (uint32_t r = 0; r < kRuns; ++r) {
                        tmem_ld_32x32b_x32(base + col(r) + 32, d1);
                        promote32(acc + r * 32, d0, r ? s1 : s0);
                        tmem_ld_wait32(d1);
                        if (r + 1 < kRuns) tmem_ld_32x32b_x32(base + col(r + 1), d0);
                        promote32(acc + r * 32 + 16, d1, r ? s1 : s0);
                        if (r + 1 < kRuns) tmem_ld_wait32(d0);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[b]);
                a0 = a1; u0 = u1; w0 = w1;
                a1 = a2; u1 = u2; w1 = w2;
            }
            if (E != EPI_SWIGLU && !alive) break;
            if constexpr (SPLIT) {
                // every copy has landed and every MMA has completed: the ring is free.
                // Partials [row][BN] fp32, 16-byte columns rotated by the row against bank conflicts.
                float4 *part = reinterpret_cast<float4 *>(smem);
                if (row_ok) {
                    const uint32_t r = quarter * 32 + lane;
#pragma unroll
                    for (uint32_t i = 0; i < kRuns * 16; ++i) {
                        const float2 x = unpack2(acc[2 * i]), y = unpack2(acc[2 * i + 1]);
                        const uint32_t c4 = half * (BN / 8) + i;
                        part[r * (BN / 4) + ((c4 + r) & (BN / 4 - 1))] = make_float4(x.x, x.y, y.x, y.y);
                    }
                }
            } else if constexpr (E == EPI_SWIGLU) {
                // mid = silu(gate) * up in fp32; one scale per row over the tile's 128
                // channels, which this thread shares with the other column half's
                float vmax = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) {
                    const float2 gt = unpack2(acc[i]), up = unpack2(acc[32 + i]);
                    float2 v;
                    v.x = __fdividef(gt.x, 1.0f + __expf(-gt.x)) * up.x;
                    v.y = __fdividef(gt.y, 1.0f + __expf(-gt.y)) * up.y;
                    vmax = fmaxf(vmax, fmaxf(fabsf(v.x), fabsf(v.y)));
                    asm("mov.b64 %0, {%1, %2};" : "=l"(acc[i]) : "f"(v.x), "f"(v.y));
                }
                const uint32_t r = quarter * 32 + lane;
                float *ax = amax_x + (n_done & 1u) * 256;   // the barrier of the tile in between orders its reuse
                ax[half * 128 + r] = vmax;
                alive = !promo_any(!alive);                 // all warps go on, or none does
                if (!alive) break;
                // below 1e-30 the group is zero for every output type; the floor keeps qmax / vmax finite
                vmax = fminf(fmaxf(fmaxf(ax[r], ax[128 + r]), 1.0e-30f), 3.0e38f);
                const float qmax = f8_max(p.out_fmt);
                const float inv = __fdiv_rn(qmax, vmax);
                if (row_ok) {
                    uint4 *o = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p.out) + (size_t)m * p.N + tl.n0 + half * 64);
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) {
                            const float2 x = unpack2(acc[8 * i + 2 * q]), y = unpack2(acc[8 * i + 2 * q + 1]);
                            w[q] = enc_f8x2(p.out_fmt, x.x * inv, x.y * inv) | enc_f8x2(p.out_fmt, y.x * inv, y.y * inv) << 16;
                        }
                        o[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (half == 0)
                        p.out_scales[(size_t)m * p.nb + tl.n0 / 128] = __fdiv_rn(vmax, qmax);
                }
            } else if (row_ok) {
#pragma unroll
                for (uint32_t r = 0; r < kRuns; ++r)
                    if (tl.n0 + col(r) < p.N) store_run(p, acc + r * 32, m, tl.n0 + col(r));
            }
        }
    }

    // ---------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        mbar_wait(drain, 0, nullptr, p.err, 0xF06);   // every issued MMA has completed
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
    if constexpr (SPLIT) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (t0 < total && !*abort) {
            const Tile tl = tile_at(p, gr, t0, kCols);
            const uint32_t rows = min(tl.m_end - tl.m0, kBM), base = smem_u32(smem);
            // the cluster's CTAs take every parts-th 16-byte column of the tile, summed in rank order
            for (uint32_t i = threadIdx.x * parts + rank; i < rows * (BN / 4); i += kThreads * parts) {
                const uint32_t r = i / (BN / 4), c4 = i % (BN / 4);
                const uint32_t c = tl.n0 + 4 * c4;
                if (c >= p.N) continue;
                const uint32_t at = base + 16 * (r * (BN / 4) + ((c4 + r) & (BN / 4 - 1)));
                float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (uint32_t q = 0; q < parts; ++q) {
                    uint32_t peer;
                    float4 v;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(q));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer));
                    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
                }
                const size_t o = (size_t)(tl.m0 + r) * p.N + c;
                if (p.out_f16) {
                    __half *d = static_cast<__half *>(p.out) + o;
                    if (p.vec && c + 4 <= p.N) {
                        *reinterpret_cast<uint2 *>(d) = make_uint2(half2_bits(s.x, s.y), half2_bits(s.z, s.w));
                    } else {
                        d[0] = __float2half_rn(s.x);
                        if (c + 1 < p.N) d[1] = __float2half_rn(s.y);
                        if (c + 2 < p.N) d[2] = __float2half_rn(s.z);
                        if (c + 3 < p.N) d[3] = __float2half_rn(s.w);
                    }
                } else {
                    float *d = static_cast<float *>(p.out) + o;
                    if (p.vec && c + 4 <= p.N) {
                        *reinterpret_cast<float4 *>(d) = s;
                    } else {
                        d[0] = s.x;
                        if (c + 1 < p.N) d[1] = s.y;
                        if (c + 2 < p.N) d[2] = s.z;
                        if (c + 3 < p.N) d[3] = s.w;
                    }
                }
            }
        }
        // a peer may still be reading this CTA's partials
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

}  // namespace fp8
}  // namespace mpp41
