"""The FP8 expert layer against 64-bit arithmetic on the same quantized weights, with
the routing that the router gives, and the router, layer and graph run together.

Tolerance, with b = 2^-4 the half step of E4M3 (2^-3 for E5M2): x is quantized
exactly as in the reference. A mid value computed in fp32 may round to the other
neighbour where it is within about 2^-20 of a midpoint, a step of 2 b |mid|; the
expected share of such values is 2^-20 / b, so flips add an error of about
2 b sqrt(2^-20 / b) = 2 sqrt(b) 2^-10 of the output's norm, below 1e-3 for both
formats; fp32 sums add (128 + I / 128) 2^-23 and an fp16 output 2^-11. The relative
Frobenius error is held to 2e-3.
"""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


def mlp64(x, g, u, d, fmt):
    gate, upv = x @ g.T, x @ u.T
    q, s = F.quant_rows(gate / (1 + np.exp(-gate)) * upv, fmt)
    return F.dequant(q, s, 1) @ d.T


def layer64(x, ids, w, ex, sh, fmt):
    q, s = F.quant_rows(x.astype(np.float64), fmt)
    xq = F.dequant(q, s, 1)
    out = mlp64(xq, *sh, fmt) if sh else np.zeros(x.shape)
    for t in range(x.shape[0]):
        for j, e in enumerate(ids[t]):
            if 0 <= e < len(ex):
                out[t] += w[t, j] * mlp64(xq[t:t + 1], *ex[e], fmt)[0]
    return out


def weights(rng, e, i, h, fmt):
    """(codes, scales) of [e, i, h] and the dequantized list."""
    codes, scales, vals = zip(*[F.random_operand(rng, i, h, fmt, 128) for _ in range(e)])
    norm = np.float32(1 / (F.QMAX[fmt] / 8 * np.sqrt(h)))
    return (torch.stack(codes).cuda(), (torch.stack(scales) * norm).cuda(), [v * np.float64(norm) for v in vals])


def setup(rng, h, i, e, shared, fmt):
    g, u, d = weights(rng, e, i, h, fmt), weights(rng, e, i, h, fmt), weights(rng, e, h, i, fmt)
    ex = list(zip(g[2], u[2], d[2]))
    dev = (g[0], g[1], u[0], u[1], d[0], d[1])
    if not shared:
        return dev, ex, None, None
    g, u, d = weights(rng, 1, shared, h, fmt), weights(rng, 1, shared, h, fmt), weights(rng, 1, h, shared, fmt)
    return dev, ex, (g[0], g[1], u[0], u[1], d[0], d[1]), (g[2][0], u[2][0], d[2][0])


@pytest.mark.parametrize("t,h,i,e,k,shared,fmt,f16", [
    (1, 256, 128, 4, 2, 0, "e4m3", True), (1, 1024, 256, 8, 8, 128, "e4m3", False), (37, 384, 256, 6, 3, 384, "e5m2", True),
    (200, 512, 128, 3, 2, 0, "e4m3", False), (300, 256, 256, 40, 4, 256, "e4m3", True), (64, 128, 128, 1, 1, 0, "e5m2", False),
    # pairs of CTAs (1024 rows an expert and more), beside a shared expert; more ids than one planning launch takes
    (1200, 256, 256, 1, 1, 128, "e4m3", True), (2100, 384, 128, 2, 2, 256, "e5m2", False), (1501, 256, 128, 5, 3, 0, "e4m3", True),
])
def test_layer(ctx, t, h, i, e, k, shared, fmt, f16):
    import mpp41
    rng = np.random.default_rng(t + h + e)
    x = rng.standard_normal((t, h)).astype(np.float16)
    dev, ex, sdev, sh = setup(rng, h, i, e, shared, fmt)
    ids = np.stack([rng.permutation(e)[:k] for _ in range(t)]).astype(np.int32)
    if t > 8:
        ids[3] = -1                       # a padded token
        ids[4, 0] = -1
        ids[5, :] = ids[5, 0]             # the same expert in every slot
        ids[-4:] = -1
    w = rng.random((t, k)).astype(np.float32)
    desc = mpp41.moe_fp8_desc(t, h, i, e, k, shared_intermediate=shared, fmt=F.FMT[fmt], out_f16=f16)
    n = mpp41.moe_fp8_scratch_bytes(desc)
    scratch = torch.full((n + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((t * h + 64,), 5.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    ctx.moe_fp8(desc, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), *dev, out, scratch,
                shared=sdev)
    ctx.synchronize()
    ref = layer64(x, ids, w.astype(np.float64), ex, sh, fmt)
    got = out.cpu().numpy().astype(np.float64)
    assert np.all(got[t * h:] == 5) and (scratch[n:] == 0xFF).all()
    got = got[: t * h].reshape(t, h)
    assert np.linalg.norm(got - ref) <= 2e-3 * np.linalg.norm(ref)
    if t > 8 and not shared:
        assert np.all(got[3] == 0)


def test_ids_beyond_the_experts_are_reported(ctx):
    import mpp41
    rng = np.random.default_rng(0)
    t, h, i, e, k = 10, 128, 128, 4, 2
    x = rng.standard_normal((t, h)).astype(np.float16)
    dev, ex, _, _ = setup(rng, h, i, e, 0, "e4m3")
    ids = rng.integers(0, e, (t, k)).astype(np.int32)
    ids[2, 1], ids[7, 0] = e, 2 ** 31 - 1
    w = rng.random((t, k)).astype(np.float32)
    desc = mpp41.moe_fp8_desc(t, h, i, e, k)
    scratch = torch.zeros(mpp41.moe_fp8_scratch_bytes(desc), dtype=torch.uint8, device="cuda")
    out = torch.zeros(t, h, device="cuda")
    ctx.moe_fp8(desc, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), *dev, out, scratch)
    with pytest.raises(mpp41.MPP41Error) as err:
        ctx.synchronize()
    assert err.value.status == mpp41.ERR_BOUNDS
    ref = layer64(x, ids, w.astype(np.float64), ex, None, "e4m3")
    assert np.linalg.norm(out.cpu().numpy() - ref) <= 2e-3 * np.linalg.norm(ref)


@pytest.mark.parametrize("t", [77, 1001])
def test_ids_and_weights_at_any_element(ctx, t):
    """Routing arrays that start on 4 bytes, not 16, and whose length no vector divides: the same bits."""
    import mpp41
    rng = np.random.default_rng(t)
    h, i, e, k = 256, 128, 5, 3
    dev, _, _, _ = setup(rng, h, i, e, 0, "e4m3")
    x = torch.from_numpy(rng.standard_normal((t, h)).astype(np.float16)).cuda()
    ids = torch.from_numpy(rng.integers(-1, e, t * k).astype(np.int32)).cuda()
    w = torch.from_numpy(rng.random(t * k).astype(np.float32)).cuda()
    desc = mpp41.moe_fp8_desc(t, h, i, e, k)
    scratch = torch.empty(mpp41.moe_fp8_scratch_bytes(desc), dtype=torch.uint8, device="cuda")
    outs = []
    for off in (0, 1, 2, 3):
        ids_at = torch.full((t * k + 8,), e + 7, dtype=torch.int32, device="cuda")
        w_at = torch.full((t * k + 8,), float("nan"), device="cuda")
        ids_at[off:off + t * k], w_at[off:off + t * k] = ids, w
        out = torch.empty(t, h, device="cuda")
        ctx.moe_fp8(desc, x, ids_at[off:], w_at[off:], *dev, out, scratch)
        ctx.synchronize()
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:]) and torch.isfinite(outs[0]).all()


def test_all_padded_gives_zeros(ctx):
    import mpp41
    rng = np.random.default_rng(1)
    dev, _, _, _ = setup(rng, 128, 128, 2, 0, "e4m3")
    desc = mpp41.moe_fp8_desc(3, 128, 128, 2, 1, out_f16=True)
    scratch = torch.full((mpp41.moe_fp8_scratch_bytes(desc),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.ones(3, 128, dtype=torch.float16, device="cuda")
    ids = torch.full((3, 1), -1, dtype=torch.int32, device="cuda")
    ctx.moe_fp8(desc, torch.randn(3, 128, device="cuda").half(), ids, torch.ones(3, 1, device="cuda"), *dev, out, scratch)
    ctx.synchronize()
    assert not out.any()


def test_quantize_route_and_layer_together(ctx):
    """fp32 weights -> quantizer -> router -> layer, eager and as a replayed graph on a side
    stream with another token's inputs, each against 64 bits."""
    import mpp41
    rng = np.random.default_rng(4)
    t, h, i, e, k = 48, 512, 256, 16, 4
    fmt = "e4m3"
    mats, vals = [], []
    for rows, cols in ((i, h), (i, h), (h, i)):
        w32 = torch.from_numpy((rng.standard_normal((e, rows, cols)) / np.sqrt(cols)).astype(np.float32)).cuda()
        q = torch.empty(e, rows, cols, dtype=torch.uint8, device="cuda")
        s = torch.empty(e, F.up(rows), F.up(cols), device="cuda")
        for j in range(e):
            ctx.quantize_weights_fp8(1, w32[j], rows, cols, q[j], s[j])
        ctx.synchronize()
        mats += [q, s]
        vals.append([F.dequant(np.repeat(F.from_fp8(q[j], fmt), 1, 0), np.repeat(s[j].cpu().numpy().astype(np.float64), 128, 0)[:rows], 1)
                     for j in range(e)])
    ex = list(zip(*vals))
    bias = (0.1 * rng.standard_normal(e)).astype(np.float32)
    x = torch.empty(t, h, dtype=torch.float16, device="cuda")
    z = torch.empty(t, e, device="cuda")
    db = torch.from_numpy(bias).cuda()
    ids, w = torch.empty(t, k, dtype=torch.int32, device="cuda"), torch.empty(t, k, device="cuda")
    gd = mpp41.gate_desc(t, e, k, score=mpp41.GATE_SIGMOID, groups=4, top_groups=2, group_top=2, scale=2.5)
    md = mpp41.moe_fp8_desc(t, h, i, e, k)
    scratch = torch.empty(mpp41.moe_fp8_scratch_bytes(md), dtype=torch.uint8, device="cuda")
    out = torch.empty(t, h, device="cuda")

    def step():
        ctx.moe_gate(gd, z, db, ids, w)
        ctx.moe_fp8(md, x, ids, w, *mats, out, scratch)

    def inputs():
        x.copy_(torch.from_numpy(rng.standard_normal((t, h)).astype(np.float16)))
        z.copy_(torch.from_numpy(rng.standard_normal((t, e)).astype(np.float32)))

    def verify():
        rid, rw = F.gate(z.cpu().numpy(), bias, k, True, 4, 2, 2, True, 2.5)
        assert np.array_equal(ids.cpu().numpy(), rid)
        ref = layer64(x.cpu().numpy(), rid, rw, ex, None, fmt)
        assert np.linalg.norm(out.cpu().numpy() - ref) <= 2e-3 * np.linalg.norm(ref)

    inputs()
    step()
    ctx.synchronize()
    verify()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    ctx.set_stream(side.cuda_stream)
    try:
        with torch.cuda.graph(g, stream=side):
            step()
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        inputs()
        g.replay()
        torch.cuda.synchronize()
        verify()
    ctx.synchronize()
