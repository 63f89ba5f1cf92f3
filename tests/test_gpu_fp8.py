"""FP8 quantizers and block-scaled products against 64-bit restatements.

Quantizers: codes and scales are equal to the definition (activations: the correctly
rounded quotient; weights: the fp32 formula), scales within half an ulp (2^-24).
Products: every fp32 operation (the tensor core's adds inside a block, taken as
truncating, 2^-23 each; the product of the scales and one fma a block) is off by at
most 2^-23 of the running sum of absolute values, so
  |error| <= (128 + K / 128 + 3) * 2^-23 * sum_k |a_k b_k|,
and fp16 results add half a step, 2^-11 |c| (2^-25 where they are subnormal).
"""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("t,h", [(1, 128), (3, 7168), (37, 4096), (5, 1), (7, 61), (4, 129), (64, 144), (2, 16), (129, 130),
                                 (1000, 256)])
def test_quantize_act(ctx, fmt, t, h):
    rng = np.random.default_rng(t + h)
    x = (rng.standard_normal((t, h)) * np.exp(rng.uniform(-12, 6, (t, 1)))).astype(np.float16)
    x[0, : min(h, 128)] = 0                                 # an all-zero block
    x[-1] = np.float16(6e-8) * rng.integers(0, 3, h)        # subnormals
    if t > 2:
        x[1] = (rng.integers(1, 15, h) * 7 / 2).astype(np.float16)   # amax a multiple of 7: exact midpoints occur
        x[1, 0] = 448 / 8
    q = torch.zeros(t * h + 64, dtype=torch.uint8, device="cuda")
    s = torch.zeros(t, F.up(h), dtype=torch.float32, device="cuda")
    ctx.quantize_act_fp8(F.FMT[fmt], torch.from_numpy(x).cuda(), t, h, q, s)
    ctx.synchronize()
    rq, rs = F.quant_rows(x.astype(np.float64), fmt)
    assert np.array_equal(F.from_fp8(q[: t * h], fmt).reshape(t, h), rq)
    assert np.all(np.abs(s.cpu().numpy() - rs) <= rs * 2.0 ** -24)
    assert not q[t * h:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_act_every_quotient(ctx, fmt):
    """All fp16 magnitudes against many block maxima: the quotient's rounding is exact, midpoints included."""
    vals = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16)
    rows = []
    for amax in [1.0, 448.0, 7.0, 3.5, 1.75, 0.875, 1.3330078125, 65504.0, 2047.0, 1792.0, 0.4375, 5.97e-8 * 7, 100.0]:
        m = np.float16(amax)
        ok = vals[vals <= m][-127 * 64:]
        ok = np.concatenate([ok, np.zeros(-len(ok) % 127, np.float16)]).reshape(-1, 127)
        rows.append(np.concatenate([np.full((len(ok), 1), m), ok], axis=1))
    x = np.concatenate(rows).astype(np.float16)
    t = len(x)
    q, s = torch.zeros(t, 128, dtype=torch.uint8, device="cuda"), torch.zeros(t, 1, device="cuda")
    ctx.quantize_act_fp8(F.FMT[fmt], torch.from_numpy(x).cuda(), t, 128, q, s)
    ctx.synchronize()
    assert np.array_equal(F.from_fp8(q, fmt), F.quant_rows(x.astype(np.float64), fmt)[0])


@pytest.mark.parametrize("h", [128, 100])
def test_quantize_act_infinities_and_nan(ctx, h):
    x = np.ones((5, h), np.float16)
    x[0, 3] = np.inf
    x[1, 4] = -np.inf
    x[2, 5] = np.nan
    x[3] = np.nan
    q, s = torch.zeros(5, h, dtype=torch.uint8, device="cuda"), torch.zeros(5, 1, device="cuda")
    ctx.quantize_act_fp8(1, torch.from_numpy(x).cuda(), 5, h, q, s)
    ctx.synchronize()
    v = F.from_fp8(q, "e4m3")
    sat = x.astype(np.float64)
    sat[0, 3], sat[1, 4] = 65504.0, -65504.0
    rq, rs = F.quant_rows(sat[:2], "e4m3")
    assert np.array_equal(v[:2], rq) and np.allclose(s.cpu().numpy()[:2], rs, rtol=2.0 ** -24)
    assert np.isnan(v[2, 5]) and np.all(np.delete(v[2], 5) == 448) and np.isnan(v[3]).all()
    assert s[2].item() == np.float32(1 / 448) and s[3].item() == 1.0


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("n,k", [(128, 128), (1, 1), (300, 512), (129, 132), (257, 333), (64, 7168), (128, 4)])
def test_quantize_weights(ctx, fmt, n, k):
    rng = np.random.default_rng(n + k)
    w = (rng.standard_normal((n, k)) * 0.02).astype(np.float32)
    w[: min(n, 128), : min(k, 128)] *= 0 if n > 200 else 1
    w[128:256, : min(k, 128)] *= np.float32(1e-36)          # maxima that qmax / amax would overflow for
    q = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    s = torch.zeros(F.up(n), F.up(k), device="cuda")
    ctx.quantize_weights_fp8(F.FMT[fmt], torch.from_numpy(w).cuda(), n, k, q, s)
    ctx.synchronize()
    pad = np.zeros((F.up(n) * 128, F.up(k) * 128), np.float32)
    pad[:n, :k] = w
    blk = pad.reshape(F.up(n), 128, F.up(k), 128)
    amax = np.abs(blk).max(axis=(1, 3))
    safe = np.where(amax > 0, amax, np.float32(1))
    by, qmax = safe[:, None, :, None], np.float32(F.QMAX[fmt])
    v = np.where(by < np.float32(1e-30), (blk / by) * qmax, blk * (qmax / np.maximum(by, np.float32(1e-30))))
    rq = F.nearest8(v.astype(np.float64), fmt).reshape(pad.shape)[:n, :k]
    assert np.array_equal(F.from_fp8(q, fmt), rq)
    assert np.array_equal(s.cpu().numpy(), np.where(amax > 0, amax / np.float32(F.QMAX[fmt]), np.float32(1)))


def product_bound(a, b, k):
    return (128 + F.up(k) + 3) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)


def check_product(got, a, b, k, f16):
    ref = a @ b.T
    tol = product_bound(a, b, k)
    if f16:
        tol = tol + np.abs(ref) * 2.0 ** -11 + 2.0 ** -25
    assert np.all(np.abs(got.astype(np.float64) - ref) <= tol)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("m,n,k", [
    (1, 128, 128), (1, 1, 16), (1, 4096, 2048), (3, 200, 144), (17, 129, 400), (32, 256, 1024), (33, 640, 512), (100, 1000, 1040),
    (128, 384, 2000), (129, 130, 256), (200, 2049, 272), (300, 512, 4096), (1000, 4096, 512), (2000, 5000, 144),
    (5, 20000, 96), (260, 19000, 160), (4, 300, 14336),
    # pairs of CTAs: the odd one without rows, without columns, with neither
    (1100, 5120, 272), (1280, 4964, 144), (1100, 4964, 528),
    # their bulk stores cut off behind the last column, in both types
    (1100, 4968, 272), (1057, 5144, 128),
])
def test_matmul(ctx, m, n, k, f16):
    rng = np.random.default_rng(m + n + k)
    fa, fb = [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")][(m + n) % 4]
    qa, sa, a = F.random_operand(rng, m, k, fa, 1)
    qb, sb, b = F.random_operand(rng, n, k, fb, 128)
    if f16:   # keep the results inside fp16
        f = np.float32(2.0 ** -np.ceil(np.log2(np.abs(a @ b.T).max() / 1000)))
        sa, a = sa * f, a * f
    dt = torch.float16 if f16 else torch.float32
    c = torch.full((m * n + 64,), 7.0, dtype=dt, device="cuda")
    ctx.matmul_fp8(F.FMT[fa], qa.cuda(), sa.cuda(), F.FMT[fb], qb.cuda(), sb.cuda(), c, m, n, k, c_f16=f16)
    ctx.synchronize()
    got = c.cpu().numpy()
    assert np.all(got[m * n:] == 7)
    check_product(got[: m * n].reshape(m, n), a, b, k, f16)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("counts,n,k,tail", [
    ([5], 256, 256, 0), ([0, 0, 3, 0], 128, 128, 2), ([128, 1, 0, 130], 200, 272, 9), ([0, 0], 64, 64, 5),
    ([300, 40, 7, 513, 1], 640, 512, 0), ([2500, 0, 700], 516, 400, 5), ([2500, 0, 700], 520, 400, 5), ([1501, 1030], 2088, 144, 3),
    ([0], 300, 128, 1100), ([5, 4000], 256, 1040, 0), ([1] * 40, 130, 144, 1), ([0] * 31 + [64] + [2] * 100, 256, 128, 3),
])
def test_grouped(ctx, counts, n, k, tail, f16):
    rng = np.random.default_rng(sum(counts) + n)
    m, groups = sum(counts) + tail, len(counts)
    qa, sa, a = F.random_operand(rng, m, k, "e4m3", 1)
    bs = [F.random_operand(rng, n, k, "e4m3", 128) for _ in counts]
    if f16:
        f = np.float32(2.0 ** -24)
        sa, a = sa * f, a * f
    off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    c = torch.full((m, n), 3.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    ctx.matmul_fp8_grouped(1, qa.cuda(), sa.cuda(), 1, torch.stack([x[0] for x in bs]).cuda(),
                           torch.stack([x[1] for x in bs]).cuda(), off, groups, c, m, n, k, c_f16=f16)
    ctx.synchronize()
    got, at = c.cpu().numpy(), 0
    for g, cnt in enumerate(counts):
        check_product(got[at:at + cnt], a[at:at + cnt], bs[g][2], k, f16)
        at += cnt
    assert np.all(got[at:] == 3)


def test_grouped_bad_offsets_are_clamped_and_reported(ctx):
    """Offsets out of order or beyond M read and write nothing outside and turn into a status."""
    import mpp41
    rng = np.random.default_rng(0)
    m, n, k = 200, 128, 128
    qa, sa, a = F.random_operand(rng, m, k, "e4m3", 1)
    qb, sb, b = F.random_operand(rng, 3 * n, k, "e4m3", 128)
    off = torch.tensor([-5, 50, 20, 100000], dtype=torch.int32, device="cuda")
    c = torch.full((m + 8, n), 3.0, device="cuda")
    ctx.matmul_fp8_grouped(1, qa.cuda(), sa.cuda(), 1, qb.cuda(), sb.cuda(), off, 3, c, m, n, k)
    with pytest.raises(mpp41.MPP41Error) as e:
        ctx.synchronize()
    assert e.value.status == mpp41.ERR_BOUNDS
    assert torch.all(c[m:] == 3)
    ctx.synchronize()


def test_matmul_special_values(ctx):
    """NaN and infinite scales stay in their rows and columns; zero scales give zeros."""
    rng = np.random.default_rng(1)
    m, n, k = 70, 300, 256
    qa, sa, _ = F.random_operand(rng, m, k, "e4m3", 1)
    qb, sb, b = F.random_operand(rng, n, k, "e4m3", 128)
    qa[3, 5] = 0x7F                     # NaN
    sa[10] = 0.0
    sa[11, 1] = float("inf")
    c = torch.zeros(m, n, device="cuda")
    ctx.matmul_fp8(1, qa.cuda(), sa.cuda(), 1, qb.cuda(), sb.cuda(), c, m, n, k)
    ctx.synchronize()
    c = c.cpu()
    assert torch.isnan(c[3]).all() and (c[10] == 0).all() and not torch.isfinite(c[11]).any()
    keep = [i for i in range(m) if i not in (3, 11)]
    assert torch.isfinite(c[keep]).all()


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (300, 1024, 512)])
def test_repeats_give_the_same_bits_and_graphs_replay(ctx, m, n, k):
    rng = np.random.default_rng(2)
    qa, sa, _ = F.random_operand(rng, m, k, "e4m3", 1)
    qb, sb, _ = F.random_operand(rng, n, k, "e4m3", 128)
    qa, sa, qb, sb = qa.cuda(), sa.cuda(), qb.cuda(), sb.cuda()
    c = [torch.zeros(m, n, device="cuda") for _ in range(3)]
    call = lambda out: ctx.matmul_fp8(1, qa, sa, 1, qb, sb, out, m, n, k)  # noqa: E731
    call(c[0])
    call(c[1])
    ctx.synchronize()
    side = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    ctx.set_stream(side.cuda_stream)
    try:
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                call(c[2])
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    c[2].zero_()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c[0], c[1]) and torch.equal(c[0], c[2])
