"""Rounding of the FP8 weight quantizer.

The codes are those of the exact quotient w * qmax / amax, rounded once.
w and amax have 24 bits and qmax = 7 * 2^n, so a quotient that is no midpoint of the 8-bit
format (at most 5 bits) is 2^-30 of its size away from it at least: 64-bit arithmetic, with
its 2^-53, decides every case.
"""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


def midpoints(fmt):
    """Positive midpoints between neighbours of the 8-bit format."""
    v = np.sort(np.abs(F.from_fp8(torch.arange(0, 0x7F if fmt == "e4m3" else 0x7C, dtype=torch.uint8), fmt)))
    return (v[1:] + v[:-1]) / 2


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("depth", [512, 511])
def test_weight_codes_next_to_midpoints(ctx, fmt, depth):
    """Values on and next to every midpoint, for many block maxima, subnormal ones among them."""
    rng = np.random.default_rng(depth)
    amax = np.concatenate([np.float32([1.0, 448.0, 3.5, 1.75, 3.4028235e38, 1e-30, 9.9e-31, 1e-37, 2e-38, 1e-41]),
                           np.exp(rng.uniform(-10, 3, 22)).astype(np.float32)])
    rows = 128 * len(amax)
    m = midpoints(fmt)
    w = np.zeros((rows, depth), np.float32)
    for i, a in enumerate(amax):
        at = (rng.choice(m, (128, depth)) * np.float64(a) / F.QMAX[fmt]).astype(np.float32)
        step = rng.integers(-2, 3, at.shape)
        near = at.view(np.int32) + np.where(at.view(np.int32) > 2, step, 0).astype(np.int32)
        at = np.minimum(near.view(np.float32), a) * rng.choice(np.float32([-1, 1]), at.shape)
        at[0, ::100] = a
        w[128 * i:128 * (i + 1)] = at
    kb = F.up(depth)
    q = torch.zeros(rows, depth, dtype=torch.uint8, device="cuda")
    s = torch.zeros(len(amax), kb, device="cuda")
    ctx.quantize_weights_fp8(F.FMT[fmt], torch.from_numpy(w).cuda(), rows, depth, q, s)
    ctx.synchronize()
    by = np.repeat(amax.astype(np.float64), 128)[:, None]
    ref = F.nearest8(w.astype(np.float64) * F.QMAX[fmt] / by, fmt)
    assert np.array_equal(F.from_fp8(q, fmt), ref)
    assert np.array_equal(s.cpu().numpy(), np.repeat((amax / np.float32(F.QMAX[fmt]))[:, None], kb, 1))
