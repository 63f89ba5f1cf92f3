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
// Warp roles (384 threads): 0 TMA producer of B, 1 MMA issuer and TMEM owner, 2 TMA
// producer of A, 3 the groups' tables (then its registers go to the promotion warps),
// 4..11 promotion (warp w: TMEM lane quarter w % 4, column half (w - 4) / 4). With one
// warp for copies and MMAs the 4096 x 14336 x 4096 product took 360 us: a block's copies
// take it as long to issue as the block's MMAs take to run. Sixteen promotion warps of
// half the columns (112 registers each) took 276 us.
//
// What bounds it: with many rows the promotion. That product takes 214 us (2.25 PFLOP/s)
// in short runs, 247 at the power limit; of 244 us in an earlier form 48 went without the FMAs, 63 without reading
// tensor memory either, 17 without the copies, and the epilogue's stores cost 20 of 230.
// With few rows it is the stream of B from memory.
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
constexpr uint32_t kBTile = 128 * kBK;      // 128 rows of B

// Shared memory of the groups' tables.
__host__ __device__ constexpr uint32_t group_bytes(uint32_t groups) { return 4 * (3 * groups + 1); }

enum Epi { EPI_STORE = 0, EPI_SWIGLU = 1 };
// SINGLE: one CTA a tile, persistent. PAIR: two CTAs of a cluster share a 256-row tile:
// tcgen05 cta_group::2 with M = 256, each CTA holding its 128 rows of A and half of B's
// columns, so a K block brings 32 KB into each SM instead of 48 KB; persistent. SPLIT:
// one tile a cluster, its CTAs take ranges of K blocks.
enum Mode { SINGLE = 0, PAIR = 1, SPLIT = 2 };

// AR: rows of A a stage has room for. With AR = 32 (at most 32 rows in the whole
// launch) the MMA still reads 128 rows from the stage's start: the other 96 come
// from the neighbouring stages and only reach accumulator lanes nobody reads.
template <int BN, int AR, int MODE> struct Cfg {
    static constexpr uint32_t kRuns = BN / 128;                     // runs of 128 columns, each with its scale of B
    static constexpr uint32_t kTileRows = MODE == PAIR ? 256 : 128;
    static constexpr uint32_t kAStage = AR * kBK;
    static constexpr uint32_t kBStage = (MODE == PAIR ? 1 : kRuns) * kBTile;   // PAIR: run `rank` only
    static constexpr int kStages = BN == 256 ? 4 : (AR == 32 ? 9 : 6);
    // PAIR: C leaves by bulk copies (store_boxes) from room that two more stages would take
    // (6, 5 and 4 stages run alike). SINGLE's stages are larger, and with three of them 32
    // groups of 512 rows took 258 us against 255, of 16 rows 77 against 75.
    static constexpr bool kBoxes = MODE == PAIR;
    static constexpr uint32_t kOutWarp = kBoxes ? 8192 : 2048;
    static constexpr uint32_t kOffB = ((kStages * kAStage + 1023) / 1024) * 1024;
    static constexpr uint32_t kOffOut = kOffB + kStages * kBStage;  // kOutWarp a promotion warp: epilogue transposition
    static constexpr uint32_t kOffAmax = kOffOut + 8 * kOutWarp;        // SwiGLU: [2 halves][128] floats
    static constexpr uint32_t kOffBar = kOffAmax + 1024;
    static constexpr uint32_t kOffGroups = kOffBar + 256;           // 3 words per group + 1
    static constexpr uint32_t kSmem = kOffGroups;                   // + group_bytes(all_groups)
    static constexpr uint32_t kAccs = 512 / BN;                     // accumulators in tensor memory, all of it
    static_assert(AR * kBK * (kStages - 1) + 128 * kBK <= kOffB + kStages * kBStage, "MMA reads stay inside the ring");
    static_assert(kSmem + group_bytes(kFp8MaxGroups + 1) <= 227 * 1024, "shared memory");
    static_assert(8 * (2 * kStages + 2 * kAccs + 1) + 8 <= 256, "barriers");
};

// One product's operands. A launch walks the tiles of two: the grouped one and, beside
// it, one more dense product (an expert layer's shared expert, whose few tiles alone
// would leave most SMs idle).
struct Side {
    CUtensorMap tm_a;           // A [M][K], box {128, box_rows}, SW128
    CUtensorMap tm_b0, tm_b1;   // B [groups * N][K], box {128, 128}, SW128 (tm_b1: the up weights, SwiGLU)
    const float *sa;            // [M][kb]
    const float *sb0, *sb1;     // [groups][nb][kb]
    void *out;                  // C [M][N], or the 8-bit mid [M][N] of the SwiGLU form
    float *out_scales;          // SwiGLU: [M][nb]
    const float *row_scale;     // factor of each row of C, or null
    uint32_t M, N, kb, nb, n_tiles;
    CUtensorMap tm_c;           // C [M][N] as bytes, box {128, 32}, SW128 (boxes)
    int vec;                    // rows of C start on 16-byte boundaries
    int boxes;                  // tm_c is made
};

struct Params {
    Side side[2];
    const int32_t *offsets;     // [groups + 1] or null (one group of all rows)
    uint32_t groups;            // of side 0; group number `groups` is side 1 where it has rows
    uint32_t all_groups;        // groups, or groups + 1
    uint32_t idesc;
    uint32_t box_rows;          // rows of A a copy brings (32 or 128)
    int out_f16;
    int out_fmt;                // SwiGLU: 8-bit format of the mid (FMT_*)
    uint32_t *err;
};

// Bounded wait of a converged warp for an mbarrier phase, with one outcome for the warp.
// The roles hand over to one another every K block, so the usual case is one poll that
// succeeds (13 cycles) and a vote (17); a try_wait with a time limit of its own takes 59,
// the limit's timer is read every 64th poll only. Two such waits at 94 cycles each paced
// the MMA issuer.
__device__ __forceinline__ bool wait_slow(uint32_t addr, uint32_t parity, volatile int *abort, uint32_t *err, uint32_t site)
{
    uint64_t t0 = 0;
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(addr, parity)) return true;
        if ((it & 63u) == 0) {
            if (*abort) return false;
            const uint64_t now = globaltimer_ns();
            if (!t0) t0 = now;
            if (now - t0 > kWaitLimitNs) {
                report_error(err, kErrTimeout, site);
                *abort = 1;
                return false;
            }
        }
    }
}

__device__ __forceinline__ bool wait_all(uint64_t *bar, uint32_t parity, volatile int *abort, uint32_t *err, uint32_t site)
{
    const uint32_t addr = smem_u32(bar);
    if (__all_sync(0xffffffffu, mbar_try_wait(addr, parity))) return true;
    return __all_sync(0xffffffffu, wait_slow(addr, parity, abort, err, site));
}

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

// ---- CTA pairs: see Mode. Barriers that the MMA issuer (even CTA) waits on live in the
// even CTA; the odd one arrives on them through shared::cluster addresses. What they
// order is copies and tensor-memory accesses (tcgen05 fences), no generic memory, so
// the arrivals and waits keep the CTA's scope: with cluster scope each one flushed
// stores or dropped L1 lines, and the 4096 x 14336 x 4096 product ran at 572 us.
__device__ __forceinline__ void mma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ uint32_t cta_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Address of the same shared-memory object in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void *local, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
    return r;
}

__device__ __forceinline__ void arrive_cl(uint32_t caddr)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(caddr) : "memory");
}

__device__ __forceinline__ void arrive_expect_tx_cl(uint32_t caddr, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(caddr), "r"(bytes) : "memory");
}

// Tiled load into this CTA's shared memory, counted on an mbarrier of either CTA of the pair (no multicast).
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const void *tmap, int32_t c0, int32_t c1, uint32_t bar_caddr)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_u32(dst)), "l"(tmap), "r"(c0), "r"(c1), "r"(bar_caddr)
        : "memory");
}

// Arrive on this barrier of both CTAs once all MMAs this thread issued before complete.
__device__ __forceinline__ void commit_pair(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 64 columns of this warp's lanes, complete, as pairs of neighbouring columns. Load, wait
// and pairing are one statement: the pairs are then the loaded registers themselves.
__device__ __forceinline__ void tmem_ld_pairs(uint32_t taddr, uint64_t (&r)[32])
{
    asm volatile("{\n\t.reg .b32 t<64>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {t0, t1, t2, t3, t4, t5, t6, t7, t8, t9, t10, t11, t12, t13, t14, t15, t16, t17, t18, t19, t20, t21, t22, t23, t24, t25, t26, t27, t28, t29, t30, t31, t32, t33, t34, t35, t36, t37, t38, t39, t40, t41, t42, t43, t44, t45, t46, t47, t48, t49, t50, t51, t52, t53, t54, t55, t56, t57, t58, t59, t60, t61, t62, t63}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {t0, t1};\n\t"
        "mov.b64 %1, {t2, t3};\n\t"
        "mov.b64 %2, {t4, t5};\n\t"
        "mov.b64 %3, {t6, t7};\n\t"
        "mov.b64 %4, {t8, t9};\n\t"
        "mov.b64 %5, {t10, t11};\n\t"
        "mov.b64 %6, {t12, t13};\n\t"
        "mov.b64 %7, {t14, t15};\n\t"
        "mov.b64 %8, {t16, t17};\n\t"
        "mov.b64 %9, {t18, t19};\n\t"
        "mov.b64 %10, {t20, t21};\n\t"
        "mov.b64 %11, {t22, t23};\n\t"
        "mov.b64 %12, {t24, t25};\n\t"
        "mov.b64 %13, {t26, t27};\n\t"
        "mov.b64 %14, {t28, t29};\n\t"
        "mov.b64 %15, {t30, t31};\n\t"
        "mov.b64 %16, {t32, t33};\n\t"
        "mov.b64 %17, {t34, t35};\n\t"
        "mov.b64 %18, {t36, t37};\n\t"
        "mov.b64 %19, {t38, t39};\n\t"
        "mov.b64 %20, {t40, t41};\n\t"
        "mov.b64 %21, {t42, t43};\n\t"
        "mov.b64 %22, {t44, t45};\n\t"
        "mov.b64 %23, {t46, t47};\n\t"
        "mov.b64 %24, {t48, t49};\n\t"
        "mov.b64 %25, {t50, t51};\n\t"
        "mov.b64 %26, {t52, t53};\n\t"
        "mov.b64 %27, {t54, t55};\n\t"
        "mov.b64 %28, {t56, t57};\n\t"
        "mov.b64 %29, {t58, t59};\n\t"
        "mov.b64 %30, {t60, t61};\n\t"
        "mov.b64 %31, {t62, t63};\n\t"
        "}"
        : "=l"(r[0]), "=l"(r[1]), "=l"(r[2]), "=l"(r[3]), "=l"(r[4]), "=l"(r[5]), "=l"(r[6]), "=l"(r[7]), "=l"(r[8]), "=l"(r[9]), "=l"(r[10]), "=l"(r[11]), "=l"(r[12]), "=l"(r[13]), "=l"(r[14]), "=l"(r[15]), "=l"(r[16]), "=l"(r[17]), "=l"(r[18]), "=l"(r[19]), "=l"(r[20]), "=l"(r[21]), "=l"(r[22]), "=l"(r[23]), "=l"(r[24]), "=l"(r[25]), "=l"(r[26]), "=l"(r[27]), "=l"(r[28]), "=l"(r[29]), "=l"(r[30]), "=l"(r[31])
        : "r"(taddr) : "memory");
}

// acc += d * s on pairs: half the instructions of scalar FMAs, which the promotion warps
// share their schedulers and instruction cache with the MMA issuer and the producers for
// (4096 x 14336 x 4096: 234 against 237 us, 32 groups of 512 rows: 273 against 280).
__device__ __forceinline__ void promote_pairs(uint64_t *acc, const uint64_t (&d)[32], uint64_t s)
{
#pragma unroll
    for (int i = 0; i < 32; ++i) asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i]) : "l"(d[i]), "l"(s));
}

__device__ __forceinline__ uint64_t dup2(float s)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(s));
    return r;
}

// g / (1 + e^-g) within 10 * 2^-24 of its size: expf (1 ulp), the sum, the reciprocal (2^-23)
// and a product; 0 below -88.7, where e^-g is infinite. Taken at a quarter of its size the
// divisor has a normal reciprocal over the whole range. (__expf is off by |g| 2^-23 more;
// a division instead of the reciprocal: 332 against 301 us for the layer of 128 tokens.)
__device__ __forceinline__ float silu(float g)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(expf(-g), 0.25f, 0.25f)));
    return 0.25f * g * r;
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
    const uint32_t *cum;    // [all_groups + 1] tiles before group g
    const uint32_t *row0;   // [all_groups]
    const uint32_t *row1;   // [all_groups]
};

struct Tile {
    uint32_t g, m0, m_end, n0, side;
};

// Tile t: groups in order; inside a group the row tile runs fastest, so that the
// CTAs of a wave share the weight tile they stream.
template <uint32_t ROWS>
__device__ __forceinline__ Tile tile_at(const Params &p, const Groups &gr, uint32_t t, uint32_t cols)
{
    uint32_t lo = 0, hi = p.all_groups;   // cum[lo] <= t < cum[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (gr.cum[mid] <= t) lo = mid; else hi = mid;
    }
    const uint32_t mt = (gr.row1[lo] - gr.row0[lo] + ROWS - 1) / ROWS, l = t - gr.cum[lo];
    Tile o;
    o.side = lo == p.groups ? 1u : 0u;
    o.g = o.side ? 0u : lo;
    o.m0 = gr.row0[lo] + (l % mt) * ROWS;
    o.m_end = gr.row1[lo];
    o.n0 = (l / mt) * cols;
    return o;
}

// Prefix sums of the groups' tiles (one warp). Offsets are clamped to [0, M] and raised to
// the largest before them: wrong ones are reported, lead nowhere out of A or C, and give
// every row to one group at most.
template <uint32_t ROWS>
__device__ __forceinline__ void build_groups(const Params &p, uint32_t *cum, uint32_t *row0, uint32_t *row1, uint32_t lane)
{
    const uint32_t per = (p.all_groups + 31) / 32;
    auto tiles = [&](uint32_t g) { return (row1[g] - row0[g] + ROWS - 1) / ROWS * p.side[g == p.groups].n_tiles; };
    uint32_t sum = 0, least = 0;   // least: the largest start of the groups before
    bool bad = false;
    if (p.offsets) {
        uint32_t most = 0;
        for (uint32_t i = 0; i < per; ++i) {
            const uint32_t g = lane * per + i;
            if (g >= p.groups) break;
            const int32_t o0 = p.offsets[g], o1 = p.offsets[g + 1], m = (int32_t)p.side[0].M;
            const int32_t a = min(max(o0, 0), m), b = min(max(o1, 0), m);
            bad |= a != o0 || b != o1;
            row0[g] = (uint32_t)a;
            row1[g] = (uint32_t)b;
            most = max(most, (uint32_t)a);
        }
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, most, o);
            if (lane >= (uint32_t)o) most = max(most, v);
        }
        least = __shfl_up_sync(0xffffffffu, most, 1);
        if (lane == 0) least = 0;
    }
    for (uint32_t i = 0; i < per; ++i) {
        const uint32_t g = lane * per + i;
        if (g >= p.all_groups) break;
        uint32_t a = 0, b = p.side[g == p.groups].M;
        if (p.offsets && g < p.groups) {
            a = max(row0[g], least);
            b = max(row1[g], a);
            bad |= a != row0[g] || b != row1[g];
            least = a;
        }
        row0[g] = a;
        row1[g] = b;
        sum += tiles(g);
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
        if (g >= p.all_groups) break;
        cum[g] = base;
        base += tiles(g);
    }
    if (lane == 31) cum[p.all_groups] = inc;
}

// ---- epilogue: 32 rows x 64 bytes of a warp through shared memory (2 KB, 16-byte units
// rotated by the row against bank conflicts), so that a store instruction covers eight
// whole 64-byte row segments instead of 32 rows' 16 bytes.
__device__ __forceinline__ uint8_t *staged(uint8_t *buf, uint32_t row, uint32_t j)
{
    return buf + row * 64 + ((j ^ (row >> 1)) & 3u) * 16;
}

__device__ __forceinline__ void stage_put(uint8_t *buf, uint32_t lane, uint32_t j, uint4 v)
{
    *reinterpret_cast<uint4 *>(staged(buf, lane, j)) = v;
}

// The staged 64 bytes of rows [m, m + 32) below m_end, at byte `off` of rows of `pitch` bytes.
__device__ __forceinline__ void stage_out(uint8_t *buf, uint32_t lane, uint8_t *out, size_t pitch, size_t off, uint32_t m, uint32_t m_end)
{
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t r = i * 8 + (lane >> 2), j = lane & 3;
        const uint4 v = *reinterpret_cast<const uint4 *>(staged(buf, r, j));
        if (m + r < m_end) *reinterpret_cast<uint4 *>(out + (size_t)(m + r) * pitch + off + j * 16) = v;
    }
    __syncwarp();
}

// 16 bytes of a row of C from column v of its 64: 8 fp16 or 4 fp32 values.
__device__ __forceinline__ uint4 unit_f16(const float *v)
{
    return make_uint4(half2_bits(v[0], v[1]), half2_bits(v[2], v[3]), half2_bits(v[4], v[5]), half2_bits(v[6], v[7]));
}

__device__ __forceinline__ uint4 unit_f32(const float *v)
{
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

// A warp's 32 rows x 64 columns of C from column c: lane = row.
__device__ __forceinline__ void store_run(const Side &p, int out_f16, const float *acc, uint8_t *buf, uint32_t lane, uint32_t m, uint32_t m_end, uint32_t c)
{
    const uint32_t size = out_f16 ? 2u : 4u;
    if (p.vec && c + 64 <= p.N) {
        uint8_t *out = static_cast<uint8_t *>(p.out);
        const size_t pitch = (size_t)p.N * size;
        if (out_f16) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) stage_put(buf, lane, j, unit_f16(acc + 32 * h + 8 * j));
                stage_out(buf, lane, out, pitch, (size_t)(c + 32 * h) * 2, m, m_end);
            }
        } else {
#pragma unroll
            for (uint32_t h = 0; h < 4; ++h) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) stage_put(buf, lane, j, unit_f32(acc + 16 * h + 4 * j));
                stage_out(buf, lane, out, pitch, (size_t)(c + 16 * h) * 4, m, m_end);
            }
        }
        return;
    }
    // rows that do not start on 16 bytes, or the last columns: 16 columns at a time
#pragma unroll
    for (uint32_t h = 0; h < 4; ++h) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            stage_put(buf, lane, j, unit_f32(acc + 16 * h + 4 * j));
        }
        __syncwarp();
        const uint32_t cc = lane & 15, col = c + 16 * h + cc;
#pragma unroll 4
        for (uint32_t i = 0; i < 16; ++i) {
            const uint32_t r = 2 * i + (lane >> 4);
            const float v = *reinterpret_cast<const float *>(staged(buf, r, cc >> 2) + (cc & 3) * 4);
            if (m + r < m_end && col < p.N) {
                const size_t at = (size_t)(m + r) * p.N + col;
                if (out_f16) static_cast<__half *>(p.out)[at] = __float2half_rn(v);
                else static_cast<float *>(p.out)[at] = v;
            }
        }
        __syncwarp();
    }
}

// The same for 32 whole rows, by bulk tensor copies that run on while the warp goes on
// (4096 x 14336 x 4096: 219.5 against 221.6 us, 4096 x 7168 x 2048 in fp32: 74.3 against
// 76.6): 128 bytes of every row (64 columns in fp16, 32 in fp32) into one of two slots, whose last
// copy has been read by then. Columns behind the last are cut off by the tensor map.
__device__ __forceinline__ void store_boxes(const Side &p, int out_f16, const float *acc, uint8_t *buf, uint32_t &boxes, uint32_t lane, uint32_t m, uint32_t c)
{
    auto slot = [&] {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        __syncwarp();
        return buf + (boxes & 1u) * 4096;
    };
    auto out = [&](const uint8_t *from, uint32_t byte) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n\t"
                         "cp.async.bulk.commit_group;"
                         ::"l"(&p.tm_c), "r"((int32_t)byte), "r"((int32_t)m), "r"(smem_u32(from))
                         : "memory");
        ++boxes;
    };
    if (out_f16) {
        uint8_t *s = slot();
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) *reinterpret_cast<uint4 *>(s + lane * 128 + ((j ^ lane) & 7u) * 16) = unit_f16(acc + 8 * j);
        out(s, c * 2);
    } else {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            if (c + 32 * h >= p.N) break;
            uint8_t *s = slot();
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                *reinterpret_cast<uint4 *>(s + lane * 128 + ((j ^ lane) & 7u) * 16) = unit_f32(acc + 32 * h + 4 * j);
            out(s, (c + 32 * h) * 4);
        }
    }
}

// SPLIT adds the CTAs' fp32 partials in rank order through distributed shared memory
// (few rows: one CTA a weight tile would leave SMs idle); nothing but C leaves the cluster.
template <int BN, int AR, int E, int MODE>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Params p)
{
    using C = Cfg<BN, AR, MODE>;
    constexpr int S = C::kStages;
    constexpr uint32_t NA = C::kAccs;
    constexpr uint32_t kRuns = C::kRuns;     // a promotion thread has 64 columns of each run
    constexpr uint32_t kCols = E == EPI_SWIGLU ? BN / 2 : BN;   // output columns per tile
    // The kernel has no static shared memory, so the dynamic part starts on its alignment.
    // Addresses are then constants: rounding the base up would cost the promotion warps
    // a register pair for every array.
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) report_error(p.err, kErrBounds, 0xF82);
        return;
    }
    uint8_t *sA = smem, *sB = smem + C::kOffB;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kOffBar);
    uint64_t *full = bars, *empty = bars + S, *acc_full = empty + S, *acc_empty = acc_full + NA, *drain = acc_empty + NA;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float *amax_x = reinterpret_cast<float *>(smem + C::kOffAmax);
    uint32_t *cum = reinterpret_cast<uint32_t *>(smem + C::kOffGroups);
    uint32_t *row0 = cum + p.all_groups + 1, *row1 = row0 + p.all_groups;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = MODE == SINGLE ? 0u : cta_rank();
    if (threadIdx.x == 0) {
        constexpr uint32_t kSides = MODE == PAIR ? 2 : 1;   // the even CTA's full / acc_empty count both CTAs
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 2 * kSides);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t b = 0; b < NA; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 8 * kSides);
        }
        mbar_init(drain, 1);
        *abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.side[0].tm_a);
        tma_prefetch_desc(&p.side[0].tm_b0);
    }
    if (warp == 1) {
        if constexpr (MODE == PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        }
    }
    // SPLIT launches are short: what is above touches no global memory and overlaps the end
    // of a kernel before that lets it. They do not let the next one start early (see
    // launch_overlapped); chains of them run no slower for it (100 x 14336 x 4096: 18.3 us,
    // 18.6 with it). Persistent launches lost 2 % to the early CTAs of the next kernel.
    if constexpr (MODE == SPLIT) pdl_wait_prior();
    if (warp == 3) build_groups<C::kTileRows>(p, cum, row0, row1, lane);
    tc_fence_before();
    __syncthreads();
    if constexpr (MODE == PAIR) cluster_sync();   // the peer's barriers are initialised before any remote arrive
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Groups gr{cum, row0, row1};

    // SPLIT: K blocks [k0, k1) of this CTA. Clusters walk the tiles.
    uint32_t t0 = blockIdx.x, step = gridDim.x, k0 = 0, parts = 1;
    if constexpr (MODE == PAIR) {
        t0 >>= 1;
        step >>= 1;
    }
    if constexpr (MODE == SPLIT) {
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
        t0 = blockIdx.x / parts;
        step = gridDim.x / parts;
        k0 = (uint32_t)((uint64_t)p.side[0].kb * rank / parts);
    }
    const uint32_t total = cum[p.all_groups];
    // end of a tile's K blocks for this CTA
    auto k_end = [&](const Side &sd) -> uint32_t {
        return MODE == SPLIT ? (uint32_t)((uint64_t)sd.kb * (rank + 1) / parts) : sd.kb;
    };

    // BN = 256: a promotion thread keeps 128 accumulators and 64 words in flight, more
    // than the 168 registers it is launched with: 128 * 40 + 256 * 232 = 384 * 168.
    if (warp < 4) {
      if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
      if (warp == 0 || warp == 2) {
        // ------------------------------------------------ TMA producers: 0 B, 2 A
        // (one warp issuing a stage's copies one after the other paces small tiles)
        const bool is_b = warp == 0;
        uint8_t *ring = is_b ? sB : sA;
        const uint32_t stage = is_b ? C::kBStage : C::kAStage;
        uint32_t st = 0, ph = 1, g = 0;
        bool alive = true;
        for (uint32_t t = t0; t < total && alive; t += step) {
            const Tile tl = tile_at<C::kTileRows>(p, gr, t, kCols);
            const Side &sd = p.side[tl.side];
            const uint32_t k1 = k_end(sd);
            // copies of this CTA for a block: row i * rows_per of its first, and how many.
            // A: its rows of the tile (none for the odd CTA of a short one). B: a copy a run;
            // the second run is the up weights, or the next 128 columns (none behind the last).
            const uint32_t m0 = tl.m0 + (MODE == PAIR ? rank * kBM : 0u), rows = m0 < tl.m_end ? min(tl.m_end - m0, kBM) : 0u;
            const bool two = kRuns == 2 && (E == EPI_SWIGLU || tl.n0 + 128 < sd.N);
            const bool first = MODE != PAIR || rank == 0, second = two && (MODE != PAIR || rank == 1);
            const uint32_t box = is_b ? 128u : p.box_rows;
            const uint32_t copies = is_b ? (first ? 1u : 0u) + (second ? 1u : 0u) : (rows + box - 1) / box;
            const CUtensorMap *tm = is_b ? (first || E != EPI_SWIGLU ? &sd.tm_b0 : &sd.tm_b1) : &sd.tm_a;
            const CUtensorMap *tm1 = is_b && E == EPI_SWIGLU ? &sd.tm_b1 : tm;
            const int32_t row = is_b ? (int32_t)(tl.g * sd.N + tl.n0) + (first || E == EPI_SWIGLU ? 0 : 128) : (int32_t)m0;
            const int32_t row_step = is_b && E == EPI_SWIGLU ? 0 : (int32_t)box;
            const uint32_t box_bytes = box * kBK, bytes = copies * box_bytes;
            for (uint32_t kk = k0; kk < k1; ++kk, ++g) {
                if (!wait_all(&empty[st], ph, abort, p.err, 0xF01)) { alive = false; break; }
                if (elect_one_sync()) {
                    const int32_t kc = (int32_t)(kk * kBK);
                    uint8_t *dst = ring + st * stage;
                    if constexpr (MODE == PAIR) {
                        const uint32_t bar = peer_addr(&full[st], 0);
                        arrive_expect_tx_cl(bar, bytes);
                        for (uint32_t i = 0; i < copies; ++i)
                            tma_load_2d_pair(dst + i * box_bytes, i ? tm1 : tm, kc, row + (int32_t)i * row_step, bar);
                    } else {
                        mbar_arrive_expect_tx(&full[st], bytes);
                        for (uint32_t i = 0; i < copies; ++i)
                            tma_load_2d(dst + i * box_bytes, i ? tm1 : tm, kc, row + (int32_t)i * row_step, &full[st]);
                    }
                }
                __syncwarp();
                if (++st == (uint32_t)S) { st = 0; ph ^= 1u; }
            }
        }
        // drain: no copy may still be landing when the CTA exits (PAIR: the even CTA's
        // barriers count both CTAs' copies, and the odd one waits for it)
        if (MODE != PAIR || rank == 0)
            for (uint32_t q = (g > (uint32_t)S ? g - S : 0); q < g; ++q)
                mbar_wait(&full[q % S], (q / S) & 1u, nullptr, p.err, 0xF02);
        // PAIR: the even CTA's commits arrive here too, the last round of them unasked for; a CTA
        // that left before they land would have them written into its successor's memory
        if (MODE == PAIR && is_b && alive)
            for (uint32_t q = (g > (uint32_t)S ? g - S : 0); q < g; ++q)
                mbar_wait(&empty[q % S], (q / S) & 1u, nullptr, p.err, 0xF07);
      } else if (warp == 1 && (MODE != PAIR || rank == 0)) {
        // ------------------------------------------------ MMA issuer
        const uint64_t ad0 = smem_desc_sw128(sA), bd0 = smem_desc_sw128(sB);
        uint32_t st = 0, ph = 0, b = 0, bph = 1;
        bool alive = true;
        for (uint32_t t = t0; t < total && alive; t += step) {
            const uint32_t k1 = k_end(p.side[p.all_groups == p.groups ? 0u : tile_at<C::kTileRows>(p, gr, t, kCols).side]);
            for (uint32_t kk = k0; kk < k1; ++kk) {
                const uint64_t ad = ad0 + st * (C::kAStage >> 4), bd = bd0 + st * (C::kBStage >> 4);
                if (!wait_all(&full[st], ph, abort, p.err, 0xF04) ||
                    !wait_all(&acc_empty[b], bph, abort, p.err, 0xF03)) { alive = false; break; }
                tc_fence_after();
                if (elect_one_sync()) {
#pragma unroll
                    for (uint32_t k = 0; k < kBK / 32; ++k) {
                        if constexpr (MODE == PAIR) mma_f8_pair(tmem + b * BN, ad + 2 * k, bd + 2 * k, p.idesc, k != 0u);
                        else mma_f8(tmem + b * BN, ad + 2 * k, bd + 2 * k, p.idesc, k != 0u);
                    }
                    if constexpr (MODE == PAIR) {
                        commit_pair(&acc_full[b]);
                        commit_pair(&empty[st]);
                    } else {
                        mma_commit(&acc_full[b]);
                        mma_commit(&empty[st]);
                    }
                }
                __syncwarp();
                if (++st == (uint32_t)S) { st = 0; ph ^= 1u; }
                if (++b == NA) { b = 0; bph ^= 1u; }
            }
        }
        if (elect_one_sync()) {
            if constexpr (MODE == PAIR) commit_pair(drain);
            else mma_commit(drain);
        }
        __syncwarp();
      }
    } else {
        if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // ------------------------------------------------ promotion and epilogue
        const uint32_t quarter = warp & 3, half = (uint32_t)(warp - 4) >> 2;
        const uint32_t lane_base = (quarter * 32u) << 16;
        uint8_t *buf = smem + C::kOffOut + (warp - 4) * C::kOutWarp;
        uint32_t boxes = 0;
        uint32_t g = 0;
        bool alive = true;
        // Scales a block ahead, and a tile's first before the epilogue of the tile before:
        // taken over at the top of the next block, when their loads have had that time
        // (the latter: 32 groups of 512 rows 259 against 268 us, 8192^3 515 against 521).
        // run r: accumulator columns [64 half, + 64) of run r's 128
        const float *sa = nullptr, *sb0 = nullptr, *sb1 = nullptr;
        float an = 0.0f, u0n = 0.0f, u1n = 0.0f;
        auto fetch = [&](uint32_t kk) {
            an = __ldg(sa + kk);
            u0n = __ldg(sb0 + kk);
            if constexpr (kRuns == 2) u1n = __ldg(sb1 + kk);
        };
        const uint32_t warp_row = (MODE == PAIR ? rank * kBM : 0u) + quarter * 32;
        auto begin = [&](uint32_t t) {
            const Tile n = tile_at<C::kTileRows>(p, gr, t, kCols);
            const Side &sd = p.side[n.side];
            const uint32_t m = n.m0 + warp_row + lane, nblk = n.n0 / 128;
            sa = sd.sa + (size_t)(m < n.m_end ? m : n.m0) * sd.kb;
            sb0 = sd.sb0 + ((size_t)n.g * sd.nb + nblk) * sd.kb;
            if (E == EPI_SWIGLU) sb1 = sd.sb1 + ((size_t)n.g * sd.nb + nblk) * sd.kb;
            else sb1 = sb0 + (kRuns == 2 && nblk + 1 < sd.nb ? sd.kb : 0u);
            fetch(k0);
            return n;
        };
        Tile next{};
        if (MODE != SPLIT && t0 < total) next = begin(t0);
        for (uint32_t t = t0; t < total && alive; t += step) {
            if (MODE == SPLIT) next = begin(t);
            const Tile tl = next;
            const Side &sd = p.side[tl.side];
            const uint32_t k1 = k_end(sd);
            const uint32_t m_warp = tl.m0 + warp_row, m = m_warp + lane;
            const bool live = m_warp < tl.m_end;   // this warp has rows
            const bool row_ok = m < tl.m_end;
            uint64_t acc2[kRuns * 32];
#pragma unroll
            for (uint32_t i = 0; i < kRuns * 32; ++i) acc2[i] = 0;
            // read out: the accumulator may be filled again
            auto release = [&](uint32_t b) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (MODE == PAIR) arrive_cl(peer_addr(&acc_empty[b], 0));
                    else mbar_arrive(&acc_empty[b]);
                }
            };
            if (live) {
                // One body, not unrolled: its code, the MMA issuer's and the producers' share
                // the instruction cache.
#pragma unroll 1
                for (uint32_t kk = k0; kk < k1; ++kk, ++g) {
                    const float s0 = an * u0n, s1 = kRuns == 2 ? an * u1n : s0;
                    if (kk + 1 < k1) fetch(kk + 1);
                    const uint32_t b = g % NA;
                    if (!wait_all(&acc_full[b], (g / NA) & 1u, abort, p.err, 0xF05)) { alive = false; break; }
                    tc_fence_after();
                    const uint32_t base = tmem + lane_base + b * BN + half * 64;
                    uint64_t d[32];
                    tmem_ld_pairs(base, d);
                    if constexpr (kRuns == 2) {
                        promote_pairs(acc2, d, dup2(s0));
                        tmem_ld_pairs(base + 128, d);
                    }
                    release(b);
                    promote_pairs(acc2 + kRuns * 32 - 32, d, dup2(s1));
                }
            } else {
                for (uint32_t kk = k0; kk < k1; ++kk, ++g) {
                    if (!wait_all(&acc_full[g % NA], (g / NA) & 1u, abort, p.err, 0xF05)) { alive = false; break; }
                    release(g % NA);
                }
            }
            if (MODE != SPLIT && t + step < total) next = begin(t + step);
            float acc[kRuns * 64];
#pragma unroll
            for (uint32_t i = 0; i < kRuns * 32; ++i) asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[2 * i]), "=f"(acc[2 * i + 1]) : "l"(acc2[i]));
            if (E != EPI_SWIGLU && !alive) break;
            if (MODE == SPLIT && parts > 1) {
                // every copy has landed and every MMA has completed: the ring is free.
                // Partials [row][BN] fp32, 16-byte columns rotated by the row against bank conflicts.
                float4 *part = reinterpret_cast<float4 *>(smem);
                if (row_ok) {
                    const uint32_t r = quarter * 32 + lane;
#pragma unroll
                    for (uint32_t i = 0; i < kRuns * 16; ++i) {
                        const uint32_t c4 = i / 16 * 32 + half * 16 + i % 16;
                        part[r * (BN / 4) + ((c4 + r) & (BN / 4 - 1))] =
                            make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
                    }
                }
            } else if (E == EPI_SWIGLU) {
                // mid = silu(gate) * up in fp32; one scale per row over the tile's 128
                // channels, which this thread shares with the other column half's
                float vmax = 0.0f;
                if (live) {
#pragma unroll
                    for (uint32_t i = 0; i < 64; ++i) {
                        acc[i] = silu(acc[i]) * acc[64 + i];
                        vmax = fmaxf(vmax, fabsf(acc[i]));
                    }
                }
                const uint32_t r = quarter * 32 + lane;
                amax_x[half * 128 + r] = vmax;
                alive = !promo_any(!alive);                 // all warps go on, or none does
                if (!alive) break;
                vmax = fmaxf(amax_x[r], amax_x[128 + r]);
                asm volatile("barrier.sync 1, %0;" ::"n"(kPromoThreads) : "memory");   // before the next tile's write
                if (live) {
                    // as the activation quantizer: scale 1 where all is zero, infinities as the largest
                    // finite value. Blocks so small that qmax / vmax would overflow are raised first.
                    vmax = fminf(vmax, 3.402823466e38f);
                    const float qmax = f8_max(p.out_fmt), raise = vmax < 0x1p-100f ? 0x1p100f : 1.0f;
                    const float inv = vmax > 0.0f ? __fdiv_rn(qmax, vmax * raise) : 0.0f;
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) {
                            const float *v = acc + 16 * i + 4 * q;
                            w[q] = enc_f8x2(p.out_fmt, v[0] * raise * inv, v[1] * raise * inv) | enc_f8x2(p.out_fmt, v[2] * raise * inv, v[3] * raise * inv) << 16;
                        }
                        stage_put(buf, lane, i, make_uint4(w[0], w[1], w[2], w[3]));
                    }
                    stage_out(buf, lane, static_cast<uint8_t *>(sd.out), sd.N, tl.n0 + half * 64, m_warp, tl.m_end);
                    if (row_ok && half == 0) sd.out_scales[(size_t)m * sd.nb + tl.n0 / 128] = vmax > 0.0f ? __fdiv_rn(vmax, qmax) : 1.0f;
                }
            } else if (live) {
                if (sd.row_scale) {
                    const float f = row_ok ? sd.row_scale[m] : 0.0f;
#pragma unroll
                    for (uint32_t i = 0; i < kRuns * 64; ++i) acc[i] *= f;
                }
                // groups end anywhere: a box that crosses the end would write the next group's rows
                const bool whole = sd.boxes && m_warp + 32 <= tl.m_end;
                if (C::kBoxes && !whole && boxes) {
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
                }
#pragma unroll
                for (uint32_t r = 0; r < kRuns; ++r) {
                    const uint32_t c = tl.n0 + r * 128 + half * 64;
                    if (c >= sd.N) break;
                    if (C::kBoxes && whole) store_boxes(sd, p.out_f16, acc + r * 64, buf, boxes, lane, m_warp, c);
                    else store_run(sd, p.out_f16, acc + r * 64, buf, lane, m_warp, tl.m_end, c);
                }
            }
        }
        if (C::kBoxes && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    // ---------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    // every issued MMA has completed (PAIR: the even CTA's last commit arrives in both)
    if (warp == 1) mbar_wait(drain, 0, nullptr, p.err, 0xF06);
    __syncthreads();
    // PAIR: neither CTA leaves while the other arrives on its barriers or the MMAs
    // read its memory. SPLIT: the partials are complete.
    if (MODE == PAIR || (MODE == SPLIT && parts > 1)) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (MODE == PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else tmem_dealloc(tmem, 512);
    }
    if (MODE == SPLIT && parts > 1) {
        if (t0 < total && !*abort) {
            const Tile tl = tile_at<C::kTileRows>(p, gr, t0, kCols);
            const Side &sd = p.side[0];
            const uint32_t rows = min(tl.m_end - tl.m0, kBM), base = smem_u32(smem);
            // the cluster's CTAs take a run of rows each, summed in rank order (interleaved
            // columns share 32-byte sectors: 100 x 4096 x 2048 10.4 against 8.4 us)
            const uint32_t i1 = rows * (rank + 1) / parts * (BN / 4);
            for (uint32_t i = rows * rank / parts * (BN / 4) + threadIdx.x; i < i1; i += kThreads) {
                const uint32_t r = i / (BN / 4), c4 = i % (BN / 4);
                const uint32_t c = tl.n0 + 4 * c4;
                if (c >= sd.N) continue;
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
                const size_t o = (size_t)(tl.m0 + r) * sd.N + c;
                if (p.out_f16) {
                    __half *d = static_cast<__half *>(sd.out) + o;
                    if (sd.vec && c + 4 <= sd.N) {
                        *reinterpret_cast<uint2 *>(d) = make_uint2(half2_bits(s.x, s.y), half2_bits(s.z, s.w));
                    } else {
                        d[0] = __float2half_rn(s.x);
                        if (c + 1 < sd.N) d[1] = __float2half_rn(s.y);
                        if (c + 2 < sd.N) d[2] = __float2half_rn(s.z);
                        if (c + 3 < sd.N) d[3] = __float2half_rn(s.w);
                    }
                } else {
                    float *d = static_cast<float *>(sd.out) + o;
                    if (sd.vec && c + 4 <= sd.N) {
                        *reinterpret_cast<float4 *>(d) = s;
                    } else {
                        d[0] = s.x;
                        if (c + 1 < sd.N) d[1] = s.y;
                        if (c + 2 < sd.N) d[2] = s.z;
                        if (c + 3 < sd.N) d[3] = s.w;
                    }
                }
            }
        }
        // a peer may still be reading this CTA's partials
        cluster_sync();
    }
}

}  // namespace fp8
}  // namespace mpp41
