"""Argument checks of the router, the FP8 quantizers, products and expert layer. They
run before the device is touched, so a zeroed stand-in for the context and made-up
addresses do: every call here is refused (or has nothing to do) and launches nothing."""
import ctypes as C

import pytest

import mpp41

CTX = C.create_string_buffer(1024)
A = 1 << 20   # an address that is aligned to anything and never read


def status(fn, *args):
    with pytest.raises(mpp41.MPP41Error) as e:
        fn(*args)
    return e.value.status


@pytest.fixture()
def ctx():
    c = mpp41.Context.__new__(mpp41.Context)
    c.h = C.addressof(CTX)
    yield c
    c.h = None


GATE = dict(tokens=4, experts=64, top_k=4)


@pytest.mark.parametrize("change,want", [
    (dict(experts=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(experts=513), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(top_k=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(top_k=33), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(experts=3), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(groups=5), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(groups=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(groups=64), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(groups=8, top_groups=9), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(groups=8, top_groups=0), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(groups=32, top_groups=1), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(group_top=3), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(group_top=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(score=2), mpp41.ERR_INVALID_ARGUMENT),
    (dict(scale=float("inf")), mpp41.ERR_INVALID_ARGUMENT), (dict(scale=float("nan")), mpp41.ERR_INVALID_ARGUMENT),
    (dict(tokens=1 << 31), mpp41.ERR_UNSUPPORTED_SHAPE),
])
def test_gate_descriptors(ctx, change, want):
    assert status(ctx.moe_gate, mpp41.gate_desc(**(GATE | change)), A, None, A, A) == want


def test_gate_buffers(ctx):
    d = mpp41.gate_desc(**GATE)
    for args in ((None, None, A, A), (A, None, None, A), (A, None, A, None), (A + 2, None, A, A), (A, A + 2, A, A), (A, None, A + 1, A)):
        assert status(ctx.moe_gate, d, *args) == mpp41.ERR_INVALID_ARGUMENT
    ctx.moe_gate(mpp41.gate_desc(0, 64, 4), None, None, None, None)   # nothing to do


def test_quantizers(ctx):
    for fn in (ctx.quantize_act_fp8, ctx.quantize_weights_fp8):
        for fmt in (0, 3, -1):
            assert status(fn, fmt, A, 4, 128, A, A) == mpp41.ERR_INVALID_ARGUMENT
        for args in ((None, 4, 128, A, A), (A, 4, 128, None, A), (A, 4, 128, A, None), (A + 1, 4, 128, A, A), (A, 4, 128, A, A + 2)):
            assert status(fn, 1, *args) == mpp41.ERR_INVALID_ARGUMENT
        fn(1, None, 0, 128, None, None)
        fn(1, None, 4, 0, None, None)
    assert status(ctx.quantize_weights_fp8, 1, A, 0xFFFFFFFF, 0xFFFFFFFF, A, A) == mpp41.ERR_UNSUPPORTED_SHAPE


@pytest.mark.parametrize("k", [0, 8, 24, 130])
def test_product_depth(ctx, k):
    assert status(ctx.matmul_fp8, 1, A, A, 1, A, A, A, 4, 4, k) == mpp41.ERR_UNSUPPORTED_SHAPE


def test_products(ctx):
    mm = ctx.matmul_fp8
    assert status(mm, 0, A, A, 1, A, A, A, 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    assert status(mm, 1, A, A, 5, A, A, A, 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    for bad in range(5):
        p = [A] * 5
        p[bad] = None
        assert status(mm, 1, p[0], p[1], 1, p[2], p[3], p[4], 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    for bad, off in ((0, 8), (1, 2), (2, 8), (3, 2), (4, 2)):
        p = [A] * 5
        p[bad] += off
        assert status(mm, 1, p[0], p[1], 1, p[2], p[3], p[4], 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    assert status(mm, 1, A, A, 1, A, A, A, 1 << 31, 4, 16) == mpp41.ERR_UNSUPPORTED_SHAPE
    assert status(mm, 1, A, A, 1, A, A, A, 4, 1 << 31, 16) == mpp41.ERR_UNSUPPORTED_SHAPE
    mm(1, None, None, 1, None, None, None, 0, 4, 16)
    mm(1, None, None, 1, None, None, None, 4, 0, 16)
    gr = ctx.matmul_fp8_grouped
    assert status(gr, 1, A, A, 1, A, A, A, 0, A, 4, 4, 16) == mpp41.ERR_UNSUPPORTED_SHAPE
    assert status(gr, 1, A, A, 1, A, A, A, 1025, A, 4, 4, 16) == mpp41.ERR_UNSUPPORTED_SHAPE
    assert status(gr, 1, A, A, 1, A, A, None, 2, A, 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    assert status(gr, 1, A, A, 1, A, A, A + 2, 2, A, 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    assert status(gr, 1, A, A, 1, A, A, A, 1024, A, 4, 1 << 22, 16) == mpp41.ERR_UNSUPPORTED_SHAPE


LAYER = dict(tokens=4, hidden=256, intermediate=128, experts=4, top_k=2)


@pytest.mark.parametrize("change,want", [
    (dict(hidden=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(hidden=200), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(intermediate=64), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(shared_intermediate=100), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(experts=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(experts=1025), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(top_k=0), mpp41.ERR_UNSUPPORTED_SHAPE), (dict(top_k=33), mpp41.ERR_UNSUPPORTED_SHAPE),
    (dict(fmt=0), mpp41.ERR_INVALID_ARGUMENT), (dict(tokens=1 << 30), mpp41.ERR_UNSUPPORTED_SHAPE),
])
def test_layer_descriptors(ctx, change, want):
    d = mpp41.moe_fp8_desc(**(LAYER | change))
    assert status(ctx.moe_fp8, d, *[A] * 9, A, A) == want
    with pytest.raises(mpp41.MPP41Error):
        mpp41.moe_fp8_scratch_bytes(d)


def test_layer_buffers(ctx):
    d = mpp41.moe_fp8_desc(**LAYER)
    for bad in range(11):
        p = [A] * 11
        p[bad] = None
        assert status(ctx.moe_fp8, d, *p) == mpp41.ERR_INVALID_ARGUMENT
    for bad, off in ((0, 16), (1, 2), (2, 2), (3, 8), (4, 2), (5, 8), (7, 8), (9, 8), (10, 128)):
        p = [A] * 11
        p[bad] += off
        assert status(ctx.moe_fp8, d, *p) == mpp41.ERR_INVALID_ARGUMENT
    sd = mpp41.moe_fp8_desc(**LAYER, shared_intermediate=128)
    assert status(ctx.moe_fp8, sd, *[A] * 11) == mpp41.ERR_INVALID_ARGUMENT
    ctx.moe_fp8(mpp41.moe_fp8_desc(**(LAYER | dict(tokens=0))), *[None] * 11)


def test_null_context():
    c = mpp41.Context.__new__(mpp41.Context)
    c.h = None
    assert status(c.moe_gate, mpp41.gate_desc(**GATE), A, None, A, A) == mpp41.ERR_INVALID_ARGUMENT
    assert status(c.matmul_fp8, 1, A, A, 1, A, A, A, 4, 4, 16) == mpp41.ERR_INVALID_ARGUMENT
    assert status(c.moe_fp8, mpp41.moe_fp8_desc(**LAYER), *[A] * 11) == mpp41.ERR_INVALID_ARGUMENT
