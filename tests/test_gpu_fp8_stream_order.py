"""Weights that the FP8 quantizer or an FP8 product writes, read by an MLP launched right behind
on the same stream. The MLP kernels start their weight stream before the kernel ahead of them
has finished where that one lets them; the results are those of a run with a synchronization
between, not those of the weights that the buffers held before."""
import numpy as np
import pytest
import torch

import fp8_data as F
import mpp41
from gpu_data import activations

pytestmark = pytest.mark.gpu


def mlp_call(ctx, kernel, t, h, i, scale):
    desc = mpp41.describe(kernel, t, h, i)
    x = torch.from_numpy(activations(t, h, scale=scale)).cuda()
    scratch = torch.empty(mpp41.scratch_bytes(desc), dtype=torch.uint8, device="cuda")

    def call(wg, wu, wd):
        out = torch.full((t, h), 7.0, device="cuda")
        ctx.mlp(desc, x, wg, wu, wd, None, None, None, scratch, out)
        return out

    return call


def close(got, ref):
    """Equal but for the order of fp32 sums over CTAs; other weights change every bit."""
    return torch.isfinite(ref).all() and torch.linalg.norm((got - ref).double()) <= 1e-5 * torch.linalg.norm(ref.double())


def check(ctx, call, produce, mats, old):
    """`produce` writes mats in each of several orders, the first matrix that the MLP reads last among them."""
    for m, o in zip(mats, old):
        m.copy_(o)
    torch.cuda.synchronize()
    stale = call(*mats)
    ctx.synchronize()
    for j in range(3):
        produce(j)
    ctx.synchronize()
    ref = call(*mats)
    ctx.synchronize()
    assert not close(stale, ref)
    for order in ((0, 1, 2), (1, 2, 0), (2, 0, 1)):
        for _ in range(4):
            for m, o in zip(mats, old):
                m.copy_(o)
            torch.cuda.synchronize()
            for j in order:
                produce(j)
            got = call(*mats)
            ctx.synchronize()
            assert close(got, ref)


@pytest.mark.parametrize("t,h,i", [(1, 1024, 4096), (128, 1024, 4096), (200, 512, 1024)])
def test_quantized_weights(ctx, t, h, i):
    rng = np.random.default_rng(t)
    shapes = ((i, h), (i, h), (h, i))
    w = [torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda() for s in shapes]
    mats = [torch.empty(s, dtype=torch.uint8, device="cuda") for s in shapes]
    scales = [torch.empty(F.up(a), F.up(b), device="cuda") for a, b in shapes]
    old = [torch.randint(0, 100, s, dtype=torch.uint8, device="cuda") for s in shapes]
    call = mlp_call(ctx, "mpp_mlp_h_fp8e4m3_f_n128", t, h, i, 1e-3)
    check(ctx, call, lambda j: ctx.quantize_weights_fp8(1, w[j], *shapes[j], mats[j], scales[j]), mats, old)


@pytest.mark.parametrize("t", [1, 64, 200])
def test_weights_of_a_split_product(ctx, t):
    rng = np.random.default_rng(t)
    h, i, k = 256, 512, 4096                     # few tiles: K is split over clusters
    shapes = ((i, h), (i, h), (h, i))
    ops = [F.random_operand(rng, a, k, "e4m3", 1)[:2] + F.random_operand(rng, b, k, "e4m3", 128)[:2] for a, b in shapes]
    ops = [(qa.cuda(), sa.cuda() * 2.0 ** -20, qb.cuda(), sb.cuda()) for qa, sa, qb, sb in ops]
    mats = [torch.empty(s, dtype=torch.float16, device="cuda") for s in shapes]
    old = [torch.randn(s, device="cuda").half() for s in shapes]
    call = mlp_call(ctx, "mpp_mlp_h_h_f_n128", t, h, i, 0.125)

    def produce(j):
        qa, sa, qb, sb = ops[j]
        ctx.matmul_fp8(1, qa, sa, 1, qb, sb, mats[j], *shapes[j], k, c_f16=True)

    check(ctx, call, produce, mats, old)
