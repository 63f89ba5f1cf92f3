"""Offsets of the grouped FP8 product that are not ascending or not within the rows: each is
clamped to [0, M] and raised to the largest before it, so the groups do not overlap, and the
call is reported. Tolerance as in the products' other tests."""
import numpy as np
import pytest
import torch

import fp8_data as F
from test_gpu_fp8 import check_product

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


def garbage(groups, m):
    rng = np.random.default_rng(groups)
    o = np.sort(rng.integers(0, m, groups + 1))
    at = rng.permutation(groups + 1)[: groups // 3]
    o[at] = rng.choice([-1, -2 ** 31, TOP, m + 1, 0, m, m // 2], len(at))
    return o.tolist()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("m,n,k,offsets", [
    (200, 128, 128, [-5, 50, 20, 100000]), (200, 300, 144, [150, 20, 180, 0, TOP]), (64, 128, 128, [-2 ** 31, -1, -1]),
    (64, 128, 128, [TOP, 0, 64]), (300, 200, 256, [0, 300, 100, 200, 300]), (150, 128, 128, [40, 30, 20, 10]),
    (2500, 520, 144, [1200, 100, 2400]), (2500, 516, 144, [0, 1300, 1100]),   # pairs of CTAs
    (700, 64, 128, garbage(40, 700)), (2000, 64, 128, garbage(100, 2000)), (900, 128, 16, garbage(33, 900)),
])
def test_bad_offsets(ctx, m, n, k, offsets, f16):
    import mpp41
    rng = np.random.default_rng(m + n)
    groups = len(offsets) - 1
    qa, sa, a = F.random_operand(rng, m, k, "e4m3", 1)
    bs = [F.random_operand(rng, n, k, "e4m3", 128) for _ in range(groups)]
    if f16:
        f = np.float32(2.0 ** -24)
        sa, a = sa * f, a * f
    start = np.maximum.accumulate(np.clip(np.array(offsets, np.int64), 0, m))
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    args = qa.cuda(), sa.cuda(), 1, torch.stack([x[0] for x in bs]).cuda(), torch.stack([x[1] for x in bs]).cuda()
    outs = []
    for _ in range(3):
        c = torch.full((m + 8, n), 3.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
        ctx.matmul_fp8_grouped(1, *args, off, groups, c, m, n, k, c_f16=f16)
        with pytest.raises(mpp41.MPP41Error) as e:
            ctx.synchronize()
        assert e.value.status == mpp41.ERR_BOUNDS
        outs.append(c)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    got = outs[0].cpu().numpy()
    for g in range(groups):
        s, t = start[g], start[g + 1]
        check_product(got[s:t], a[s:t], bs[g][2], k, f16)
    assert np.all(got[: start[0]] == 3) and np.all(got[start[-1]:] == 3)
    ctx.synchronize()
