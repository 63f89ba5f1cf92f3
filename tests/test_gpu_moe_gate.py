"""Expert routing against its definition in 64 bits, one token after the other.

Ids are equal. Weights: a score has expf's error (2 ulp), an addition, a division
(half an ulp each) and the argument's rounding |z| * 2^-24; with the sum, the last
division and the factor of a renormalised weight that stays below 2^-24 * (16 + 4 |z|)
relative, |z| <= 24 here: 2^-24 * 112 < 8e-6; values below 1e-37 may be lost.
"""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


def run(ctx, z, bias, k, sigmoid=True, groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0):
    import mpp41
    t, e = z.shape
    dz = torch.from_numpy(z).cuda()
    db = None if bias is None else torch.from_numpy(np.asarray(bias, np.float32)).cuda()
    ids = torch.full((t, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((t, k), -7.0, dtype=torch.float32, device="cuda")
    d = mpp41.gate_desc(t, e, k, score=mpp41.GATE_SIGMOID if sigmoid else mpp41.GATE_SOFTMAX, groups=groups,
                        top_groups=top_groups, group_top=group_top, renormalize=renorm, scale=scale,
                        logits_f16=z.dtype == np.float16)
    ctx.moe_gate(d, dz, db, ids, w)
    ctx.synchronize()
    return ids.cpu().numpy(), w.cpu().numpy().astype(np.float64)


def check(ctx, z, bias, k, **kw):
    full = dict(sigmoid=True, groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0) | kw
    ids, w = run(ctx, z, bias, k, **full)
    rid, rw = F.gate(z, bias, k, **full)
    assert np.array_equal(ids, rid), np.argwhere((ids != rid).any(axis=1))[:4].ravel()
    assert np.all(np.abs(w - rw) <= 8e-6 * np.abs(rw) + 1e-37)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("t,e,k,groups,top_groups,group_top", [
    (1, 256, 8, 8, 4, 2), (37, 256, 8, 8, 4, 2), (300, 64, 6, 1, 1, 1), (5, 1, 1, 1, 1, 1), (33, 7, 7, 7, 7, 1),
    (64, 60, 4, 5, 2, 1), (64, 60, 4, 5, 2, 2), (17, 512, 16, 16, 3, 2), (9, 160, 6, 8, 3, 1), (12, 500, 32, 4, 1, 2),
    (40, 32, 2, 32, 5, 2), (257, 129, 9, 3, 2, 2),
])
def test_gate(ctx, t, e, k, groups, top_groups, group_top, sigmoid, renorm):
    rng = np.random.default_rng(t * 1000 + e)
    z = (rng.standard_normal((t, e)) * 2).astype(np.float32)
    kw = dict(sigmoid=sigmoid, groups=groups, top_groups=top_groups, group_top=group_top, renorm=renorm, scale=2.5)
    check(ctx, z, (0.2 * rng.standard_normal(e)).astype(np.float32), k, **kw)
    check(ctx, z, None, k, **kw)
    check(ctx, z.astype(np.float16), None, k, **kw)      # fp16 logits: many exact ties


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("group_top", [1, 2])
def test_near_ties_are_decided_exactly(ctx, sigmoid, group_top):
    """Scores that agree in fp32 and differ in 64 bits, at every cut: saturated sigmoids,
    neighbouring logits, biases that differ by an ulp."""
    rng = np.random.default_rng(5)
    e = 64
    z = np.empty((6, e), np.float32)
    z[0] = 18.0 + rng.permutation(e) * 1e-3            # sigmoid rounds to 1 in fp32
    z[1] = np.float32(0.5)
    z[1, 40:] = np.nextafter(np.float32(0.5), np.float32(1))
    z[2] = 0.0                                         # exact ties: lowest indices
    z[3] = rng.permutation(e) * 1e-7
    z[4] = -20.0 - rng.permutation(e) * 1e-3
    z[5] = np.where(rng.random(e) < 0.5, 1.0, np.nextafter(np.float32(1), np.float32(2)))
    for bias in (np.zeros(e, np.float32), np.full(e, 0.25, np.float32), (rng.permutation(e) * 2.0 ** -24).astype(np.float32)):
        for groups, tg in ((1, 1), (8, 3)):
            check(ctx, z, bias, 8, sigmoid=sigmoid, groups=groups, top_groups=tg, group_top=group_top)
        check(ctx, z, None, 8, sigmoid=sigmoid, groups=8, top_groups=3, group_top=group_top)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("biased", [True, False])
def test_masks(ctx, sigmoid, renorm, biased):
    """-inf and NaN mask; a wholly masked token gets weights 0; infinities, the type's
    lowest value and huge logits stay finite."""
    rng = np.random.default_rng(9)
    e, k = 48, 6
    z = rng.standard_normal((12, e)).astype(np.float32)
    z[0] = -np.inf
    z[1] = np.nan
    z[2, 3:] = -np.inf                    # three left, six wanted
    z[3, ::2] = np.nan
    z[4] = np.finfo(np.float32).min       # the lowest finite value is no mask
    z[5, 7] = np.inf
    z[6, 5] = z[6, 40] = np.inf
    z[7] = -np.inf
    z[7, 47] = -3.0
    z[8] = 1e4 * rng.standard_normal(e)
    z[9, :24] = -np.inf                   # groups 0..3 masked
    z[10] = np.float32(-0.0)
    z[10, ::3] = np.float32(0.0)          # equal: -0 is no lower
    z[11] = np.finfo(np.float32).max
    bias = (0.3 * rng.standard_normal(e)).astype(np.float32) if biased else None
    for groups, tg, gt in ((1, 1, 1), (8, 3, 2), (8, 2, 1)):
        kw = dict(sigmoid=sigmoid, groups=groups, top_groups=tg, group_top=gt, renorm=renorm)
        ids, w = run(ctx, z, bias, k, **kw)
        rid, rw = F.gate(z, bias, k, sigmoid=sigmoid, groups=groups, top_groups=tg, group_top=gt, renorm=renorm, scale=1.0)
        assert np.array_equal(ids, rid)
        assert np.all(np.isfinite(w)) and np.all(w[0] == 0) and np.all(w[1] == 0)
        fine = np.arange(12) != 8         # logits of 1e4: the argument's rounding is 1e4 * 2^-24 of a score's logarithm
        assert np.all(np.abs(w - rw)[fine] <= 8e-6 * np.abs(rw)[fine] + 1e-37)
        assert np.all(np.abs(w - rw)[8] <= 2e-3 * np.abs(rw)[8] + 1e-37)


def test_bias_of_any_size(ctx):
    """The bias decides the choice and never enters a weight; infinite and NaN ones too."""
    rng = np.random.default_rng(3)
    z = rng.standard_normal((20, 96)).astype(np.float32)
    b = (1e6 * rng.standard_normal(96)).astype(np.float32)
    check(ctx, z, b, 5)
    b[7], b[8], b[9] = np.inf, -np.inf, np.nan
    check(ctx, z, b, 32)
    check(ctx, z, b, 20, groups=4, top_groups=3, group_top=2)


@pytest.mark.parametrize("z0", [-90.0, -200.0])
def test_tiny_scores_keep_their_ratio(ctx, z0):
    z = (z0 + np.arange(16, dtype=np.float32))[None].repeat(2, 0)
    for sigmoid in (True, False):
        check(ctx, z, None, 4, sigmoid=sigmoid)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("e,k,groups,top_groups,group_top", [
    (64, 6, 1, 1, 1), (64, 8, 4, 2, 2), (40, 5, 5, 3, 1), (7, 3, 1, 1, 1), (129, 9, 1, 1, 1),
])
def test_many_tokens(ctx, e, k, groups, top_groups, group_top, sigmoid, renorm):
    """From the token counts of a long prefill on, a warp weighs several tokens' choices
    together: a ragged last batch, ties, masks and near ties among its tokens."""
    t = 148 * 64 + 7
    rng = np.random.default_rng(e)
    z = (rng.standard_normal((t, e)) * 2).astype(np.float32)
    z[5] = 0.0
    z[6] = -np.inf
    z[7] = np.nan
    z[8, 1:] = -np.inf
    z[9] = 18.0 + rng.permutation(e) * 1e-3
    z[10] = rng.permutation(e) * 1e-7
    z[-1] = np.inf
    kw = dict(sigmoid=sigmoid, groups=groups, top_groups=top_groups, group_top=group_top, renorm=renorm, scale=2.5)
    check(ctx, z, (0.2 * rng.standard_normal(e)).astype(np.float32), k, **kw)
    check(ctx, z, None, k, **kw)
    check(ctx, z.astype(np.float16), None, k, **kw)
