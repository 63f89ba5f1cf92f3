// C ABI of the expert router, the FP8 quantizers, the block-scaled FP8 products and
// the FP8 expert layer (include/mpp41.h).
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>

#include "../../include/mpp41.h"
#include "mpp41_internal.h"

using namespace mpp41;

namespace {

constexpr uint64_t kIndexLimit = 1ull << 31;   // TMA coordinates and grid sizes are 32-bit signed

mpp41_status invalid(const char *msg) { return set_last_error(MPP41_ERR_INVALID_ARGUMENT, msg); }
mpp41_status shape(const char *msg) { return set_last_error(MPP41_ERR_UNSUPPORTED_SHAPE, msg); }

mpp41_status cuda_status(cudaError_t e, const char *what)
{
    if (e == cudaSuccess) return MPP41_OK;
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
    return set_last_error(MPP41_ERR_CUDA, buf);
}

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool fmt_ok(int f) { return f == 1 || f == 2; }
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// The context's device is current inside a call, whatever the caller's is.
struct OnDevice {
    int was = -1;
    bool ok = true;
    explicit OnDevice(int dev)
    {
        int cur = -1;
        ok = cudaGetDevice(&cur) == cudaSuccess;
        if (ok && cur != dev) {
            ok = cudaSetDevice(dev) == cudaSuccess;
            was = cur;
        }
    }
    ~OnDevice() { if (was >= 0) cudaSetDevice(was); }
};

// Arguments are checked before the device is touched.
#define NEED(ctx) \
    if (!(ctx)) return invalid("null context")
#define ON_DEVICE(ctx)                  \
    OnDevice on_device_((ctx)->device); \
    if (!on_device_.ok) return set_last_error(MPP41_ERR_CUDA, "cannot use the context's device")

mpp41_status run_gemm(const Fp8Launch &L, cudaStream_t st, const char *what)
{
    const char *why = "";
    const int rc = launch_fp8_gemm(L, st, &why);
    if (!rc) return MPP41_OK;
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", what, why);
    return set_last_error(rc == 1 ? MPP41_ERR_UNSUPPORTED_SHAPE : MPP41_ERR_CUDA, buf);
}

mpp41_status check_gemm(int a_fmt, int b_fmt, uint32_t M, uint64_t b_rows, uint32_t K)
{
    if (!fmt_ok(a_fmt) || !fmt_ok(b_fmt)) return invalid("formats must be 1 (E4M3) or 2 (E5M2)");
    if (!K || K % 16) return shape("depth must be a positive multiple of 16");
    if (M >= kIndexLimit || b_rows >= kIndexLimit || K >= kIndexLimit) return shape("sizes must be below 2^31");
    return MPP41_OK;
}

}  // namespace

extern "C" {

mpp41_status mpp41_moe_gate(mpp41_ctx *ctx, const mpp41_gate_desc *d, const void *logits, const float *bias, int32_t *ids,
                            float *weights)
{
    NEED(ctx);
    if (!d) return invalid("null gate descriptor");
    if (d->score != MPP41_GATE_SOFTMAX && d->score != MPP41_GATE_SIGMOID) return invalid("unknown score function");
    if (!d->experts || d->experts > 512) return shape("experts must be in [1, 512]");
    if (!d->groups || d->groups > 32 || d->experts % d->groups) return shape("groups must be in [1, 32] and divide experts");
    if (!d->top_groups || d->top_groups > d->groups) return shape("top_groups must be in [1, groups]");
    if (d->group_top != 1 && d->group_top != 2) return shape("group_top must be 1 or 2");
    if (!d->top_k || d->top_k > 32 || d->top_k > d->experts / d->groups * d->top_groups)
        return shape("top_k must be in [1, 32] and at most the experts of the chosen groups");
    if (!std::isfinite(d->scale)) return invalid("scale must be finite");
    if (d->tokens >= kIndexLimit) return shape("sizes must be below 2^31");
    if (!d->tokens) return MPP41_OK;
    if (!logits || !ids || !weights) return invalid("null buffer");
    if (!aligned(logits, d->logits_f16 ? 2 : 4) || !aligned(bias, 4) || !aligned(ids, 4) || !aligned(weights, 4))
        return invalid("buffers must be aligned to their elements");
    ON_DEVICE(ctx);
    GateLaunch L{logits, bias, ids, weights, d->tokens, d->experts, d->top_k, d->groups, d->top_groups, d->group_top,
                 d->score == MPP41_GATE_SIGMOID, d->renormalize != 0, d->logits_f16 != 0, d->scale};
    return cuda_status(launch_moe_gate(L, ctx->stream), "gate");
}

mpp41_status mpp41_quantize_act_fp8(mpp41_ctx *ctx, int fmt, const void *x, uint32_t tokens, uint32_t hidden, uint8_t *q,
                                    float *scales)
{
    NEED(ctx);
    if (!fmt_ok(fmt)) return invalid("format must be 1 (E4M3) or 2 (E5M2)");
    if (!tokens || !hidden) return MPP41_OK;
    if (!x || !q || !scales) return invalid("null buffer");
    if (!aligned(x, 2) || !aligned(scales, 4)) return invalid("buffers must be aligned to their elements");
    ON_DEVICE(ctx);
    return cuda_status(launch_quantize_act_fp8(fmt, x, tokens, hidden, q, scales, ctx->stream), "quantize activations");
}

mpp41_status mpp41_quantize_weights_fp8(mpp41_ctx *ctx, int fmt, const float *w, uint32_t rows, uint32_t depth, uint8_t *q,
                                        float *scales)
{
    NEED(ctx);
    if (!fmt_ok(fmt)) return invalid("format must be 1 (E4M3) or 2 (E5M2)");
    if (!rows || !depth) return MPP41_OK;
    if (((uint64_t)rows + 127) / 128 * (((uint64_t)depth + 127) / 128) >= kIndexLimit) return shape("too many blocks");
    if (!w || !q || !scales) return invalid("null buffer");
    if (!aligned(w, 4) || !aligned(scales, 4)) return invalid("buffers must be aligned to their elements");
    ON_DEVICE(ctx);
    return cuda_status(launch_quantize_weights_fp8(fmt, w, rows, depth, q, scales, ctx->stream), "quantize weights");
}

mpp41_status mpp41_matmul_fp8(mpp41_ctx *ctx, int a_fmt, const void *a, const float *sa, int b_fmt, const void *b,
                              const float *sb, void *c, uint32_t M, uint32_t N, uint32_t K, int c_f16)
{
    return mpp41_matmul_fp8_grouped(ctx, a_fmt, a, sa, b_fmt, b, sb, nullptr, 1, c, M, N, K, c_f16);
}

mpp41_status mpp41_matmul_fp8_grouped(mpp41_ctx *ctx, int a_fmt, const void *a, const float *sa, int b_fmt, const void *b,
                                      const float *sb, const int32_t *offsets, uint32_t groups, void *c, uint32_t M,
                                      uint32_t N, uint32_t K, int c_f16)
{
    NEED(ctx);
    const mpp41_status s = check_gemm(a_fmt, b_fmt, M, (uint64_t)groups * N, K);
    if (s != MPP41_OK) return s;
    if (!groups || groups > kFp8MaxGroups) return shape("groups must be in [1, 1024]");
    if (!offsets && groups != 1) return invalid("several groups need offsets");
    if (!M || !N) return MPP41_OK;
    if (!a || !sa || !b || !sb || !c) return invalid("null buffer");
    if (!aligned(a, 16) || !aligned(b, 16)) return invalid("a and b must be 16-byte aligned");
    if (!aligned(sa, 4) || !aligned(sb, 4) || !aligned(offsets, 4) || !aligned(c, c_f16 ? 2 : 4))
        return invalid("buffers must be aligned to their elements");
    ON_DEVICE(ctx);
    Fp8Launch L{};
    L.a = a; L.sa = sa; L.b0 = b; L.sb0 = sb;
    L.offsets = offsets;
    L.out = c;
    L.M = M; L.N = N; L.K = K; L.groups = groups;
    L.a_fmt = a_fmt; L.b_fmt = b_fmt;
    L.out_f16 = c_f16 != 0;
    L.err = ctx->err;
    return run_gemm(L, ctx->stream, "FP8 product");
}

}  // extern "C"

// ------------------------------------------------------------------ the expert layer
namespace {

struct MoeFp8Layout {
    size_t offsets, inv, rw, pq, ps, mq, ms, y, xq, xs, smq, sms, sy, total;
};

MoeFp8Layout moe_fp8_layout(const mpp41_moe_fp8_desc *d)
{
    const size_t T = d->tokens, H = d->hidden, I = d->intermediate, R = T * d->top_k, Is = d->shared_intermediate;
    const size_t Ts = Is ? T : 0;
    MoeFp8Layout l;
    size_t o = 0;
    auto part = [&](size_t bytes) { const size_t at = o; o += up256(bytes); return at; };
    l.offsets = part((d->experts + (size_t)1) * 4);
    l.inv = part(R * 4);
    l.rw = part(R * 4);
    l.pq = part(R * H);
    l.ps = part(R * (H / 128) * 4);
    l.mq = part(R * I);
    l.ms = part(R * (I / 128) * 4);
    l.y = part(R * H * 4);
    l.xq = part(Ts * H);
    l.xs = part(Ts * (H / 128) * 4);
    l.smq = part(Ts * Is);
    l.sms = part(Ts * (Is / 128) * 4);
    l.sy = part(Ts * H * 4);
    l.total = o;
    return l;
}

mpp41_status check_moe_fp8(const mpp41_moe_fp8_desc *d)
{
    if (!d) return invalid("null MoE descriptor");
    if (!fmt_ok(d->fmt)) return invalid("format must be 1 (E4M3) or 2 (E5M2)");
    if (!d->hidden || d->hidden % 128 || !d->intermediate || d->intermediate % 128 || d->shared_intermediate % 128)
        return shape("hidden and intermediate sizes must be positive multiples of 128");
    if (!d->experts || d->experts > kFp8MaxGroups) return shape("experts must be in [1, 1024]");
    if (!d->top_k || d->top_k > 32) return shape("top_k must be in [1, 32]");
    if ((uint64_t)d->tokens * d->top_k >= kIndexLimit || (uint64_t)d->experts * d->intermediate >= kIndexLimit ||
        (uint64_t)d->experts * d->hidden >= kIndexLimit || d->shared_intermediate >= kIndexLimit)
        return shape("sizes must be below 2^31");
    return MPP41_OK;
}

}  // namespace

extern "C" {

size_t mpp41_moe_fp8_scratch_bytes(const mpp41_moe_fp8_desc *d)
{
    return check_moe_fp8(d) == MPP41_OK ? moe_fp8_layout(d).total : 0;
}

mpp41_status mpp41_moe_fp8(mpp41_ctx *ctx, const mpp41_moe_fp8_desc *d, const void *x, const int32_t *ids,
                           const float *weights, const void *wg, const float *sg, const void *wu, const float *su,
                           const void *wd, const float *sd, const void *shared_wg, const float *shared_sg,
                           const void *shared_wu, const float *shared_su, const void *shared_wd, const float *shared_sd,
                           void *out, void *scratch)
{
    NEED(ctx);
    mpp41_status s = check_moe_fp8(d);
    if (s != MPP41_OK) return s;
    if (!d->tokens) return MPP41_OK;
    if (!x || !ids || !weights || !wg || !sg || !wu || !su || !wd || !sd || !out || !scratch) return invalid("null buffer");
    const uint32_t T = d->tokens, H = d->hidden, I = d->intermediate, E = d->experts, k = d->top_k, R = T * k;
    const uint32_t Is = d->shared_intermediate;
    if (Is && (!shared_wg || !shared_sg || !shared_wu || !shared_su || !shared_wd || !shared_sd))
        return invalid("shared expert weights missing");
    if (!aligned(wg, 16) || !aligned(wu, 16) || !aligned(wd, 16) || !aligned(out, 16) || !aligned(x, 32) ||
        !aligned(scratch, 256) || (Is && (!aligned(shared_wg, 16) || !aligned(shared_wu, 16) || !aligned(shared_wd, 16))))
        return invalid("weights and out must be 16-byte aligned, x 32-byte, scratch 256-byte");
    if (!aligned(ids, 4) || !aligned(weights, 4) || !aligned(sg, 4) || !aligned(su, 4) || !aligned(sd, 4) ||
        !aligned(shared_sg, 4) || !aligned(shared_su, 4) || !aligned(shared_sd, 4))
        return invalid("buffers must be aligned to their elements");
    ON_DEVICE(ctx);
    const MoeFp8Layout l = moe_fp8_layout(d);
    uint8_t *b = static_cast<uint8_t *>(scratch);
    auto f32 = [&](size_t at) { return reinterpret_cast<float *>(b + at); };
    int32_t *offsets = reinterpret_cast<int32_t *>(b + l.offsets), *inv = reinterpret_cast<int32_t *>(b + l.inv);
    cudaStream_t st = ctx->stream;
    s = cuda_status(launch_fp8_scatter(d->fmt, ids, weights, E, offsets, inv, f32(l.rw), ctx->err, x, T, H, k, b + l.pq, f32(l.ps),
                                       Is ? b + l.xq : nullptr, Is ? f32(l.xs) : nullptr, st), "plan and quantize x");
    if (s != MPP41_OK) return s;
    Fp8Launch g{}, gs{}, n{}, ns{};
    g.a = b + l.pq; g.sa = f32(l.ps);
    g.b0 = wg; g.sb0 = sg; g.b1 = wu; g.sb1 = su;
    g.offsets = offsets; g.groups = E;
    g.out = b + l.mq; g.out_scales = f32(l.ms);
    g.M = R; g.N = I; g.K = H;
    g.a_fmt = g.b_fmt = g.out_fmt = d->fmt;
    g.err = ctx->err;
    n = g;
    n.a = b + l.mq; n.sa = f32(l.ms);
    n.b0 = wd; n.sb0 = sd; n.b1 = nullptr; n.sb1 = nullptr;
    n.out = b + l.y; n.out_scales = nullptr;
    n.row_scale = f32(l.rw);
    n.N = H; n.K = I;
    if (Is) {
        gs = g;
        gs.a = b + l.xq; gs.sa = f32(l.xs);
        gs.b0 = shared_wg; gs.sb0 = shared_sg; gs.b1 = shared_wu; gs.sb1 = shared_su;
        gs.offsets = nullptr; gs.groups = 1;
        gs.out = b + l.smq; gs.out_scales = f32(l.sms);
        gs.M = T; gs.N = Is;
        ns = n;
        ns.a = b + l.smq; ns.sa = f32(l.sms);
        ns.b0 = shared_wd; ns.sb0 = shared_sd;
        ns.offsets = nullptr; ns.groups = 1;
        ns.out = b + l.sy; ns.row_scale = nullptr;
        ns.M = T; ns.K = Is;
        g.more = &gs;
        n.more = &ns;
    }
    s = run_gemm(g, st, "expert gate/up product");
    if (s != MPP41_OK) return s;
    s = run_gemm(n, st, "expert down product");
    if (s != MPP41_OK) return s;
    return cuda_status(launch_fp8_combine(f32(l.y), inv, T, k, H, Is ? f32(l.sy) : nullptr, out, d->out_f16 != 0, st), "combine");
}

}  // extern "C"
