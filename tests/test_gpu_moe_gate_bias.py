"""Group choice of the router under biases of opposite signs, against the definition in 64 bits.

A group's worth is the sum of its two best values. Where those have opposite signs the
sum is small and the roundings of its addends are not: they are as large as 2^-24 of the
bias. The choice is that of the 64-bit values all the same, so ids are equal; weights
have the tolerance of the router's other tests.
"""
import numpy as np
import pytest

import fp8_data as F
from test_gpu_moe_gate import check, run

pytestmark = pytest.mark.gpu


def test_two_groups_that_fp32_sums_order_wrongly(ctx):
    """Worths 0.84939641 and 0.84939652; summed in fp32 the first comes out 1.2e-6 larger."""
    z = np.array([[-0.60188931, -0.01806114, -0.51503229, -0.09855192]], np.float32)
    b = np.array([16.0, -16.0, 0.0, 0.0], np.float32)
    ids, _ = run(ctx, z, b, 2, groups=2, top_groups=1, group_top=2)
    assert sorted(ids[0].tolist()) == [2, 3]


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("size", [2, 4, 6])
@pytest.mark.parametrize("b", [16.0, 100.0, 1000.0, 1e6])
def test_biases_of_opposite_signs(ctx, b, size, sigmoid):
    """Groups of two, of four (on lane borders) and of six (not): their two best are +b and -b or nearly."""
    rng = np.random.default_rng(int(b) + size)
    groups = 8
    bias = np.full((groups, size), -20.0 * b)
    for g in range(groups):
        at = rng.permutation(size)
        bias[g, at[0]], bias[g, at[1]] = b * (g + 1), -b * (g + 1)
        if g < 3:
            bias[g, at[:2]] = 0.25, -0.25       # some whose values are small
    z = (rng.standard_normal((3000, groups * size)) * 2).astype(np.float32)
    for top_groups in (1, 4):
        check(ctx, z, bias.reshape(-1).astype(np.float32), 2, sigmoid=sigmoid, groups=groups, top_groups=top_groups, group_top=2)


@pytest.mark.parametrize("size", [4, 6])
@pytest.mark.parametrize("top_groups", [1, 2, 5])
def test_infinite_values_of_both_signs_in_a_group(ctx, size, top_groups):
    """+inf beside -inf is the worth -inf, behind all finite ones; +inf beside a finite value comes first."""
    rng = np.random.default_rng(size)
    groups, t = 8, 64
    z = rng.standard_normal((t, groups * size)).astype(np.float32)
    bias = (0.2 * rng.standard_normal((groups, size))).astype(np.float32)
    bias[2, 1] = np.inf
    bias[5, 0], bias[5, 1:] = np.inf, -np.inf
    z[::2, 2 * size:3 * size] = -np.inf
    z[::2, 2 * size + 1] = 0.5                   # group 2: one open expert, of value +inf
    z[1::4, 7 * size:] = np.nan                  # group 7 masked
    ids, w = run(ctx, z, bias.reshape(-1), 3, groups=groups, top_groups=top_groups, group_top=2)
    with np.errstate(invalid="ignore"):
        rid, rw = F.gate(z, bias.reshape(-1), 3, True, groups, top_groups, 2, True, 1.0)
    assert np.array_equal(ids, rid)
    assert np.all(np.abs(w - rw) <= 8e-6 * np.abs(rw) + 1e-37)
