"""Dropout with one value per plane, at plane sizes from two elements to more than a block takes, with whole and broken
groups of four planes: bit for bit the stored-mask form's values."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib
from .gpu_util import Dev, call

pytestmark = pytest.mark.gpu
F = C.c_float
SEED, FIRST = 0x0123456789ABCDEF, (1 << 32) - 3           # (the counter passes 32 bits within most of the calls)


@pytest.mark.parametrize("planes,hw", [(1, 2), (2, 2), (5, 3), (1000, 2), (4097, 3), (40, 25), (513, 49), (37, 121), (64, 1024), (3, 4096), (7, 5000), (2, 70001), (9, 16384),
                                       (3001, 4), (601, 36), (6, 1), (8, 8)])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_planes(gpu_ctx, oracle32, planes, hw, shift, p):
    rng = np.random.default_rng(planes + hw)
    total = planes * hw
    mask = np.repeat(oracle32.dropout_mask(planes, p, SEED, FIRST), hw)
    pad, end = np.zeros(shift, np.float32), np.full(8, 7.0, np.float32)
    x, r, old = (rng.standard_normal(total).astype(np.float32) for _ in range(3))
    at = lambda d: C.c_void_p(d.ptr.value + 4 * shift)
    src, res = Dev(gpu_ctx, np.concatenate([pad, x])), Dev(gpu_ctx, np.concatenate([pad, r]))

    def out(v=None):
        return Dev(gpu_ctx, np.concatenate([pad, np.full(total, np.nan, np.float32) if v is None else v, end]))

    def body(d):
        v = d.get()
        assert (v[:shift] == 0).all() and (v[shift + total:] == 7).all()
        return v[shift:shift + total]

    y = out()
    call(gpu_ctx, "nrs_dropout_fwd", at(src), None, at(y), total, hw, F(p), SEED, FIRST)
    assert np.array_equal(body(y), x * mask)
    y = out()
    call(gpu_ctx, "nrs_dropout_bwd", at(src), at(y), total, hw, F(p), SEED, FIRST, 0)
    assert np.array_equal(body(y), x * mask)
    y = out()                                             # a product and a sum, rounded once or twice
    call(gpu_ctx, "nrs_dropout_fwd", at(src), at(res), at(y), total, hw, F(p), SEED, FIRST)
    want = r.astype(np.float64) + x.astype(np.float64) * mask
    assert (np.abs(body(y) - want) <= 2.0 ** -24 * (np.abs(want) + np.abs(x * mask)) * 1.0001).all()
    y, z = out(old), out(old)
    call(gpu_ctx, "nrs_dropout_bwd", at(src), at(y), total, hw, F(p), SEED, FIRST, 1)
    call(gpu_ctx, "nrs_mask_mul", at(src), Dev(gpu_ctx, oracle32.dropout_mask(planes, p, SEED, FIRST)), at(z), total, hw, 1)
    assert np.array_equal(body(y), body(z)) or hw == 1
    z = out(x)                                            # in place
    call(gpu_ctx, "nrs_dropout_fwd", at(z), None, at(z), total, hw, F(p), SEED, FIRST)
    assert np.array_equal(body(z), x * mask)


def test_planes_past_32_bits(gpu_ctx, oracle32):
    """Three planes whose elements, and whose vectors' first elements among four planes, pass 32 bits."""
    hw = (1 << 30) + 1
    n = 3 * hw
    mask = oracle32.dropout_mask(3, 0.5, SEED, 6)
    assert len(set(mask.tolist())) == 2                   # (dropped and kept ones among them)
    x, l = Dev(gpu_ctx, shape=(n,), zero=True), _lib.lib()
    ones = np.ones(64, np.float32)
    spots = [0, hw - 32, 2 * hw - 32, n - 64]
    at = lambda i: C.c_void_p(x.ptr.value + 4 * i)
    for i in spots:
        _lib.check(gpu_ctx.h, l.nrs_h2d(gpu_ctx.h, at(i), C.c_void_p(ones.ctypes.data), ones.nbytes))
    call(gpu_ctx, "nrs_dropout_fwd", x, None, x, n, hw, F(0.5), SEED, 6)
    for i in spots:
        got = np.empty(64, np.float32)
        _lib.check(gpu_ctx.h, l.nrs_d2h(gpu_ctx.h, C.c_void_p(got.ctypes.data), at(i), got.nbytes))
        assert np.array_equal(got, mask[(i + np.arange(64)) // hw]), i
