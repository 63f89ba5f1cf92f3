"""The mid of the FP8 expert layer, silu(gate) * up in fp32, over the range of its arguments."""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


def mid_through_layer(ctx, gate, up_scale, fmt="e4m3"):
    """silu(g) * u of the layer for fp32 gates g that reach it exactly, u = 448 * 56 * 2^k.

    The token has one value, 56, in column 0: its quantized value is exact. A block's 128 channels have the same weights, so every mid is its block's maximum, has the code qmax
    and comes back as qmax * scale; the down weights add one channel, times 1."""
    import mpp41
    n = len(gate)
    h = i = 128 * n
    x = np.zeros((1, h), np.float16)
    x[0, 0] = 56
    code = lambda v: F.to_fp8(v, fmt)  # noqa: E731
    wg, wu = np.zeros((i, h)), np.zeros((i, h))
    wg[:, 0], wu[:, 0] = 1, 448
    sg, su = np.ones((n, n), np.float32), np.ones((n, n), np.float32)
    sg[:, 0] = gate / np.float32(56)
    su[:, 0] = up_scale
    wd = np.zeros((h, i))
    wd[np.arange(n) * 128, np.arange(n) * 128] = 1
    sd = np.ones((n, n), np.float32)
    dev = [torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v.cuda() for v in (code(wg), sg, code(wu), su, code(wd), sd)]
    d = mpp41.moe_fp8_desc(1, h, i, 1, 1, fmt=F.FMT[fmt])
    scratch = torch.empty(mpp41.moe_fp8_scratch_bytes(d), dtype=torch.uint8, device="cuda")
    out = torch.empty(h, device="cuda")
    ctx.moe_fp8(d, torch.from_numpy(x).cuda(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda"),
                *dev, out, scratch)
    ctx.synchronize()
    g = 56.0 * (gate / np.float32(56)).astype(np.float64)        # what the layer sums: one product, rounded
    g = g.astype(np.float32).astype(np.float64)
    u = (np.float64(56 * 448) * np.float32(up_scale)).astype(np.float32).astype(np.float64)
    return out.cpu().numpy()[::128][:n], g / (1 + np.exp(-g)) * u


@pytest.mark.parametrize("lo,hi,up", [(-60.0, -20.0, 1.0), (-20.0, 20.0, 1.0), (20.0, 80.0, 0.5), (-88.6, -87.4, 2.0 ** 60),
                                      (-80.0, -70.0, 2.0 ** -14)])
def test_mid_in_fp32(ctx, lo, hi, up):
    """expf within 1 ulp (2^-23), a reciprocal (2^-23), the sum 1 + e, the products with g and u, the
    scale, and the down product's two roundings within half an ulp each (2^-24): 10 * 2^-24, second
    order terms well below 2^-24 more. The last range has mids below 1e-30."""
    rng = np.random.default_rng(int(hi) + 100)
    got, ref = mid_through_layer(ctx, rng.uniform(lo, hi, 20).astype(np.float32), np.float32(up))
    assert np.all(np.abs(got - ref) <= 11 * 2.0 ** -24 * np.abs(ref))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_mid_of_infinities_and_zeros(ctx, fmt):
    """An infinite mid counts as the largest finite value, a block of zeros gives zeros."""
    gate = np.float32([1e30, 0.0, -200.0, 1.0])
    got, ref = mid_through_layer(ctx, gate, np.float32(2.0 ** 100), fmt)
    most = np.finfo(np.float32).max
    assert got[0] >= most * (1 - 2.0 ** -22) and got[1] == 0 and got[2] == 0
    assert abs(got[3] - ref[3]) <= 11 * 2.0 ** -24 * abs(ref[3])
