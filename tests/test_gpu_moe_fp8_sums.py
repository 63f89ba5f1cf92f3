"""Sums of the FP8 expert layer's rows where their terms cancel.

Two terms come from the same gate and up weights and from down weights of opposite
sign, so the rows y and -y have the same bits but for the sign, roundings of the mid
among them, and the layer's sum is (w0 - w1) y + the rest. fp32 rows and sums are off
by 2^-24 of each term, of which there are at most 3 here, twice each (row and sum): 6 *
2^-24 |w0 y|. With |w0 - w1| = 2^-8 |w0| that is 6 * 2^-16 of the result. y itself is held
to the 2e-3 (Frobenius) of the layer's other tests, derived there; an fp16 result adds
2^-11. Rows in fp16 would put 2^-11 / 2^-8 = 1 / 8 there, or infinities.
"""
import numpy as np
import pytest
import torch

import fp8_data as F
from test_gpu_moe_fp8 import layer64, weights

pytestmark = pytest.mark.gpu

TOL = 2e-3 + 6 * 2.0 ** -16 + 2.0 ** -11


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("partner", ["expert", "shared"])
@pytest.mark.parametrize("t", [1, 40, 300])
def test_cancelling_rows(ctx, t, partner, f16):
    import mpp41
    rng = np.random.default_rng(t)
    h, i = 256, 128
    x = rng.standard_normal((t, h)).astype(np.float16)
    g, u, d = weights(rng, 1, i, h, "e4m3"), weights(rng, 1, i, h, "e4m3"), weights(rng, 1, h, i, "e4m3")
    # rows of up to 2^18 or so, far beyond fp16's 65504; the sum is a 256th of that
    q, s = F.quant_rows(x.astype(np.float64), "e4m3")
    mid = F.dequant(q, s, 1) @ g[2][0].T
    mid = mid / (1 + np.exp(-mid)) * (F.dequant(q, s, 1) @ u[2][0].T)
    up = np.float32(2.0 ** np.floor(18 - np.log2(np.abs(mid @ d[2][0].T).max())))
    ds, dv = d[1] * up, [v * np.float64(up) for v in d[2]]
    neg = (d[0] ^ 0x80, ds, [-v for v in dv])
    w0 = rng.uniform(0.5, 1.0, t).astype(np.float32)
    small = np.float32(1 - 2.0 ** -8)
    if partner == "expert":
        gate, gs, upw, us = (v.repeat(2, 1, 1) for v in (g[0], g[1], u[0], u[1]))
        dev = (gate, gs, upw, us, torch.cat([d[0], neg[0]]), torch.cat([ds, neg[1]]))
        ids = np.tile(np.array([[0, 1]], np.int32), (t, 1))
        w = np.stack([w0, w0 * small], axis=1)
        ex, sh, sdev = [(g[2][0], u[2][0], dv[0]), (g[2][0], u[2][0], neg[2][0])], None, None
    else:
        dev = (g[0], g[1], u[0], u[1], neg[0], neg[1])
        ids, w = np.zeros((t, 1), np.int32), np.full((t, 1), small, np.float32)
        ex, sh, sdev = [(g[2][0], u[2][0], neg[2][0])], (g[2][0], u[2][0], dv[0]), (g[0], g[1], u[0], u[1], d[0], ds)
    desc = mpp41.moe_fp8_desc(t, h, i, len(ex), w.shape[1], shared_intermediate=i if sh else 0, out_f16=f16)
    scratch = torch.full((mpp41.moe_fp8_scratch_bytes(desc),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((t, h), 5.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    ctx.moe_fp8(desc, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), *dev, out, scratch,
                shared=sdev)
    ctx.synchronize()
    ref = layer64(x, ids, w.astype(np.float64), ex, sh, "e4m3")
    got = out.cpu().numpy().astype(np.float64)
    assert np.abs(ref).max() < 60000 and np.isfinite(got).all()
    assert np.linalg.norm(got - ref) <= TOL * np.linalg.norm(ref)
