"""FP8 quantizers at sides of almost 2^32 (up to 26 GB on the device)."""
import numpy as np
import pytest
import torch

import fp8_data as F

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_returned():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("hidden", [2 ** 32 - 16, 2 ** 32 - 1])
def test_quantize_act_of_the_widest_row(ctx, fmt, hidden):
    """One row of almost 2^32 values: its first and last blocks and its scales."""
    x = torch.zeros(hidden, dtype=torch.float16, device="cuda")
    ends = torch.cat([torch.arange(256), torch.arange(hidden - 300, hidden)])
    vals = torch.randn(556, generator=torch.Generator().manual_seed(1)).half()
    x[ends.cuda()] = vals.cuda()
    q = torch.full((hidden,), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((F.up(hidden),), -1.0, device="cuda")
    ctx.quantize_act_fp8(F.FMT[fmt], x, 1, hidden, q, s)
    ctx.synchronize()
    for at in (0, (hidden - 300) // 128 * 128):
        part = x[at:at + 600].cpu().numpy().astype(np.float64)[None]
        part = part[:, :256] if at == 0 else part
        rq, rs = F.quant_rows(part, fmt)
        n = part.shape[1]
        assert np.array_equal(F.from_fp8(q[at:at + n], fmt), rq[0])
        assert np.all(np.abs(s[at // 128:at // 128 + F.up(n)].cpu().numpy() - rs[0]) <= rs[0] * 2.0 ** -24)
    assert not q[256:hidden - 300].any() and (s[2:-4] == 1).all()


@pytest.mark.parametrize("rows,depth", [(1, 2 ** 32 - 4), (1, 2 ** 32 - 1), (2 ** 32 - 3, 1)])
def test_quantize_weights_of_the_longest_side(ctx, rows, depth):
    n = rows * depth
    w = torch.zeros(n, device="cuda")
    w[:2], w[-3:] = torch.tensor([1.0, 0.5]), torch.tensor([0.5, -2.0, 1.0])
    q = torch.full((n,), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((F.up(n),), -1.0, device="cuda")
    ctx.quantize_weights_fp8(1, w, rows, depth, q, s)
    ctx.synchronize()
    assert F.from_fp8(q[:2], "e4m3").tolist() == [448, 224] and F.from_fp8(q[-3:], "e4m3").tolist() == [112, -448, 224]
    assert not q[2:-3].any()
    want = np.float32([1, 2]) / np.float32(448)
    assert s[0].item() == want[0] and s[-1].item() == want[1] and (s[1:-1] == 1).all()


@pytest.mark.parametrize("f16", [True, False])
def test_layer_of_more_columns_than_the_grid_has(ctx, f16):
    """Hidden size above 2^25: the rows' sums take more CTAs than one grid dimension has. One
    expert and a shared one, whose mid is 448 in channel 0 and whose down weights are zero but
    for a few columns at both ends and beside the limit."""
    import mpp41
    h, i, k = 2 ** 25 + 256, 128, 2
    x = torch.zeros(1, h, dtype=torch.float16, device="cuda")
    x[0, 0] = 448
    one = int(F.to_fp8([1.0], "e4m3")[0])
    zeros = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
    wg, wu, wd = zeros(1, i, h), zeros(1, i, h), zeros(1, h, i)
    wg[0, 0, 0] = wu[0, 0, 0] = one
    at = torch.tensor([0, 1, 127, 2 ** 24, 2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1, h - 1], device="cuda")
    wd[0, at, 0] = one
    sg, sd = torch.full((1, 1, h // 128), 2.0 ** -4, device="cuda"), torch.full((1, h // 128, 1), 2.0 ** -6, device="cuda")
    # gate = up = 448 / 16 = 28: silu(28) * 28 = 784, and 784 / 64 = 12.25 from each of the three
    d = mpp41.moe_fp8_desc(1, h, i, 1, k, shared_intermediate=i, out_f16=f16)
    scratch = torch.empty(mpp41.moe_fp8_scratch_bytes(d), dtype=torch.uint8, device="cuda")
    out = torch.full((1, h), 5.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    ctx.moe_fp8(d, x, torch.zeros(1, k, dtype=torch.int32, device="cuda"), torch.tensor([[1.0, -3.0]], device="cuda"), wg, sg, wu,
                sg, wd, sd, out, scratch, shared=(wg, sg, wu, sg, wd, sd))
    ctx.synchronize()
    assert torch.all((out[0, at].double() + 12.25).abs() <= 12.25 * 2.0 ** -11 + 1e-5)
    out[0, at] = 0
    assert not out.any()
