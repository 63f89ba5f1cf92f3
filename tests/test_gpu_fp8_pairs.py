"""FP8 products of CTA pairs among other kernels that take over their SMs at once.

The last arrivals that a pair's even CTA sends to the odd one have landed before that one
leaves, so nothing of them reaches a successor: a run of pair products with short split
products, quantizers and a second stream between them leaves the same bits as each alone.
"""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


def test_pairs_among_other_kernels(ctx):
    import mpp41
    rng = np.random.default_rng(11)
    # rows of more than 1024 a group: pairs; the odd CTA with rows, with one, without any
    cases = [(1280, 4964, 144), (1153, 5120, 272), (1100, 4968, 528)]
    small = (16, 512, 2048)
    made = {}
    for m, n, k in cases + [small]:
        qa, sa, _ = F.random_operand(rng, m, k, "e4m3", 1)
        qb, sb, _ = F.random_operand(rng, n, k, "e4m3", 128)
        made[m, n, k] = (qa.cuda(), sa.cuda(), qb.cuda(), sb.cuda())
    x = torch.from_numpy(rng.standard_normal((64, 4096)).astype(np.float16)).cuda()

    def product(c, dims, out):
        qa, sa, qb, sb = made[dims]
        c.matmul_fp8(1, qa, sa, 1, qb, sb, out, *dims)

    def quantize(c, q, s):
        c.quantize_act_fp8(1, x, 64, 4096, q, s)

    new = lambda dims: torch.full(dims[:2], 7.0, device="cuda")  # noqa: E731
    codes = lambda: (torch.zeros(64, 4096, dtype=torch.uint8, device="cuda"), torch.zeros(64, 32, device="cuda"))  # noqa: E731
    alone = {d: new(d) for d in made}
    q0, s0 = codes()
    for d in made:
        product(ctx, d, alone[d])
        ctx.synchronize()
    quantize(ctx, q0, s0)
    ctx.synchronize()
    side = torch.cuda.Stream()
    other = mpp41.Context(0)
    other.set_stream(side.cuda_stream)
    torch.cuda.synchronize()
    work = [(c, d, new(d), new(small), codes()) for _ in range(8) for d in cases for c in (ctx, other)]
    torch.cuda.synchronize()
    for c, d, o, p, (q, s) in work:     # both streams hold work at once
        product(c, d, o)
        product(c, small, p)
        quantize(c, q, s)
    torch.cuda.synchronize()
    ctx.synchronize()
    other.synchronize()
    other.close()
    for _, d, o, p, (q, s) in work:
        assert torch.equal(o, alone[d]) and torch.equal(p, alone[small])
        assert torch.equal(q, q0) and torch.equal(s, s0)
