"""Dropout whose mask is made again in each pass: bit for bit the values of the stored-mask form, which the CPU restatement
of the counter stream pins, at every layout, alignment and length; draws as arguments; refusals."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib, cuda
from neuralrs_b200.cuda import Node, backward_graph, graph, nn
from neuralrs_b200.cuda import runtime as gpu
from .gpu_util import Dev, call

F = C.c_float
SEED, FIRST = 0xFEDCBA9876543210, (1 << 35) + 7


def off(d, floats):
    """A pointer some floats into a buffer."""
    return C.c_void_p(d.ptr.value + 4 * floats)


@pytest.mark.gpu
@pytest.mark.parametrize("total,hw", [(1, 1), (3, 1), (4, 1), (1023, 1), (4096, 1), (1_000_003, 1), (8 * 16 * 49, 49), (6 * 64, 64), (10 * 12, 12), (7, 7)])
@pytest.mark.parametrize("shift", [0, 1])
def test_forward_and_backward_are_the_stored_masks(gpu_ctx, oracle32, total, hw, shift):
    rng = np.random.default_rng(total + hw)
    p = 0.3
    mask = np.repeat(oracle32.dropout_mask(total // hw, p, SEED, FIRST), hw)
    pad = np.zeros(shift, np.float32)
    x, r, g, old = (rng.standard_normal(total).astype(np.float32) for _ in range(4))
    dx, dr, dg = (Dev(gpu_ctx, np.concatenate([pad, v])) for v in (x, r, g))
    y = Dev(gpu_ctx, np.full(total + shift + 4, 7.0, np.float32))
    call(gpu_ctx, "nrs_dropout_fwd", off(dx, shift), None, off(y, shift), total, hw, F(p), SEED, FIRST)
    got = y.get()
    assert np.array_equal(got[shift:shift + total], x * mask)
    assert (got[:shift] == 7).all() and (got[shift + total:] == 7).all()          # nothing beside it is touched
    call(gpu_ctx, "nrs_dropout_fwd", off(dx, shift), off(dr, shift), off(y, shift), total, hw, F(p), SEED, FIRST)
    want = r.astype(np.float64) + x.astype(np.float64) * mask.astype(np.float64)  # one rounding, or two
    assert (np.abs(y.get()[shift:shift + total] - want) <= 2.0 ** -24 * (np.abs(want) + np.abs(x * mask)) * 1.0001).all()
    d = Dev(gpu_ctx, np.concatenate([pad, old]))
    call(gpu_ctx, "nrs_dropout_bwd", off(dg, shift), off(d, shift), total, hw, F(p), SEED, FIRST, 0)
    assert np.array_equal(d.get()[shift:], g * mask)
    # adding: exactly what the stored-mask pass adds
    a, b = Dev(gpu_ctx, np.concatenate([pad, old])), Dev(gpu_ctx, np.concatenate([pad, old]))
    call(gpu_ctx, "nrs_dropout_bwd", off(dg, shift), off(a, shift), total, hw, F(p), SEED, FIRST, 1)
    m = Dev(gpu_ctx, oracle32.dropout_mask(total // hw, p, SEED, FIRST))
    call(gpu_ctx, "nrs_mask_mul", off(dg, shift), m, off(b, shift), total, hw, 1)
    assert np.array_equal(a.get(), b.get())


@pytest.mark.gpu
def test_in_place_and_special_values(gpu_ctx, oracle32):
    n = 4096
    x = np.linspace(-2, 2, n, dtype=np.float32)
    x[::97], x[1::97], x[2::97] = np.inf, np.nan, -np.inf
    for p in (0.0, 0.5, 1.0):
        with np.errstate(all="ignore"):
            want = x * oracle32.dropout_mask(n, p, 3, 0)
        d = Dev(gpu_ctx, x)
        call(gpu_ctx, "nrs_dropout_fwd", d, None, d, n, 1, F(p), 3, 0)
        assert np.array_equal(d.get(), want, equal_nan=True)
    r = np.arange(n, dtype=np.float32)
    d, t = Dev(gpu_ctx, np.ones(n, np.float32)), Dev(gpu_ctx, r)
    call(gpu_ctx, "nrs_dropout_fwd", d, t, t, n, 1, F(0.5), 3, 0)                  # onto the residual
    assert np.array_equal(t.get(), r + oracle32.dropout_mask(n, 0.5, 3, 0))


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu_ctx, oracle32):
    """More than 2^32 bytes of data, and a counter that crosses 32 bits inside the call."""
    n, first = (1 << 30) + 5, (1 << 32) - 9
    x = Dev(gpu_ctx, shape=(n,), zero=True)
    l = _lib.lib()
    head, tail = np.ones(64, np.float32), np.ones(69, np.float32)
    _lib.check(gpu_ctx.h, l.nrs_h2d(gpu_ctx.h, x.ptr, C.c_void_p(head.ctypes.data), head.nbytes))
    _lib.check(gpu_ctx.h, l.nrs_h2d(gpu_ctx.h, off(x, n - 69), C.c_void_p(tail.ctypes.data), tail.nbytes))
    call(gpu_ctx, "nrs_dropout_fwd", x, None, x, n, 1, F(0.5), 11, first)
    a, b = np.empty(64, np.float32), np.empty(69, np.float32)
    _lib.check(gpu_ctx.h, l.nrs_d2h(gpu_ctx.h, C.c_void_p(a.ctypes.data), x.ptr, a.nbytes))
    _lib.check(gpu_ctx.h, l.nrs_d2h(gpu_ctx.h, C.c_void_p(b.ctypes.data), off(x, n - 69), b.nbytes))
    assert np.array_equal(a, oracle32.dropout_mask(64, 0.5, 11, first))
    assert np.array_equal(b, oracle32.dropout_mask(69, 0.5, 11, first + (n - 69) // 4))


@pytest.mark.gpu
def test_take_is_the_streams_own_window(gpu_ctx):
    l = _lib.lib()
    _lib.check(gpu_ctx.h, l.nrs_rng_seed(gpu_ctx.h, 77))
    seed, first, at = C.c_uint64(), C.c_uint64(), C.c_uint64()
    for count, want in ((10, 0), (1, 3), (0, 4), (4, 4)):
        _lib.check(gpu_ctx.h, l.nrs_rng_take(gpu_ctx.h, count, C.byref(seed), C.byref(first)))
        assert (seed.value, first.value) == (77, want)
    _lib.check(gpu_ctx.h, l.nrs_rng_offset(gpu_ctx.h, C.byref(at)))
    assert at.value == 5


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(7,), (3, 5, 8), (2, 130, 64)])
def test_residual_node(gpu_ctx, oracle32, shape):
    rng = np.random.default_rng(1)
    l = _lib.lib()
    x, r, g = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
    n = x.size
    _lib.check(gpu_ctx.h, l.nrs_rng_seed(gpu_ctx.h, 5))
    nx, nr = Node.new(x, shape), Node.new(r, shape)
    for v in (nx, nr):
        gpu.to_cuda(v)
    first = nn.dropout(nx, 0.25, True)                                            # takes the stream's first blocks
    out = nn.dropout_add(first, nr, 0.25, True)
    m1, m2 = oracle32.dropout_mask(n, 0.25, 5, 0), oracle32.dropout_mask(n, 0.25, 5, (n + 3) // 4)
    h = x.ravel() * m1
    want = r.ravel().astype(np.float64) + h.astype(np.float64) * m2
    assert (np.abs(gpu.to_host(out) - want) <= 2.0 ** -24 * (np.abs(want) + np.abs(h * m2)) * 1.0001).all()
    gpu.set_grad(out, g)
    backward_graph(out)
    assert np.array_equal(gpu.read_grad(nr), g.ravel())
    assert np.array_equal(gpu.read_grad(nx), g.ravel() * m2 * m1)
    assert np.array_equal(gpu.to_host(nn.dropout_add(nx, nr, 0.25, False)), (x + r).ravel())
    # the same node twice
    _lib.check(gpu_ctx.h, l.nrs_rng_seed(gpu_ctx.h, 5))
    twice = nn.dropout_add(nr, nr, 0.25, True)
    gpu.zero_grad([nr])
    gpu.set_grad(twice, g)
    backward_graph(twice)
    want = g.ravel().astype(np.float64) * (1.0 + m1.astype(np.float64))
    assert (np.abs(gpu.read_grad(nr) - want) <= 2.0 ** -23 * np.abs(want)).all()
    with pytest.raises(_lib.NrsError):
        nn.dropout_add(nx, Node.new(np.zeros(n + 1, np.float32), [n + 1]), 0.25, True)
    with pytest.raises(_lib.NrsError):
        nn.dropout_add(nx, nr, 1.5, True)


@pytest.mark.gpu
def test_refusals(gpu_ctx):
    d = Dev(gpu_ctx, shape=(16,), zero=True)
    for args, code in [((d, None, d, 16, 1, F(1.5), 0, 0), 1), ((d, None, d, 16, 1, F(float("nan")), 0, 0), 1), ((d, None, d, 16, 0, F(0.5), 0, 0), 2),
                       ((d, None, d, 16, 3, F(0.5), 0, 0), 2), ((None, None, d, 16, 1, F(0.5), 0, 0), 1), ((d, None, None, 16, 1, F(0.5), 0, 0), 1)]:
        with pytest.raises(_lib.NrsError) as e:
            call(gpu_ctx, "nrs_dropout_fwd", *args)
        assert e.value.code == code
    call(gpu_ctx, "nrs_dropout_fwd", None, None, None, 0, 1, F(0.5), 0, 0)        # nothing to do
    call(gpu_ctx, "nrs_dropout_bwd", None, None, 0, 1, F(0.5), 0, 0, 1)


def test_null_context_is_refused(nrs_lib):
    assert nrs_lib.nrs_dropout_fwd(None, None, None, None, 0, 1, F(0.5), 0, 0) == 1
    assert nrs_lib.nrs_dropout_bwd(None, None, None, 0, 1, F(0.5), 0, 0, 0) == 1
    assert nrs_lib.nrs_rng_take(None, 1, None, None) == 1
