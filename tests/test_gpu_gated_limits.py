"""Gated feed-forward layers at the limits of what they are given: matrices of very different magnitudes side by side, gates far from
zero.  Against the formulas in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib
from .conftest import rel_l2
from .gpu_util import Dev, call

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GELU, SILU = 2, 3


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-v))


def act(a, kind):
    """act(a) and its slope without a cancellation; and the sigmoid's argument."""
    a = np.asarray(a, np.float64)
    w = a if kind == SILU else 2 * 0.7978845608 * (a + 0.044715 * a ** 3)
    dw = 1.0 if kind == SILU else 2 * 0.7978845608 * (1 + 3 * 0.044715 * a * a)
    s, r = sigmoid(w), sigmoid(-w)                        # (1 - s, to its own last bit)
    return a * s, s + np.where(s * r > 0, a * (s * r) * dw, 0.0), w

def inputs(rng, m, n, k):
    s = 1 / np.sqrt(k)
    return [v.astype(np.float32) for v in (rng.standard_normal((m, k)), rng.standard_normal((k, n)) * s, rng.standard_normal((k, n)) * s, rng.standard_normal((m, n)))]


def formulas(x, wg, wu, dh, a, u):
    """The gradients for projections a and u as they were kept (SiLU)."""
    x, wg, wu, dh, a, u = (v.astype(np.float64) for v in (x, wg, wu, dh, a, u))
    f, d, _ = act(a, SILU)
    da, du = dh * u * d, dh * f
    return dict(dx=da @ wg.T + du @ wu.T, dwg=x.T @ da, dwu=x.T @ du)


def backward(ctx, x, wg, wu, a, u, dh):
    (m, k), n = x.shape, wg.shape[1]
    out = [Dev(ctx, np.full_like(v, np.nan)) for v in (x, wg, wu)]
    call(ctx, "nrs_gated_linear_bwd", *(Dev(ctx, v) for v in (x, wg, wu, a, u, dh)), *out, m, n, k, SILU, 0, 0)
    return dict(zip(("dx", "dwg", "dwu"), (o.get() for o in out)))


# Chains of 256 values of a UMMA's truncated sums, and the operands' two roundings (tests/test_gpu_gated.py counts the same):
# whatever the other matrix is.
SHAPES = [(64, 64, 64), (200, 100, 136), (300, 260, 520), (700, 320, 96)]
LEVELS = [2.0 ** -40, 2.0 ** -90, 2.0 ** 40]


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("which", ["gate", "up"])
def test_a_weight_far_below_the_other(gpu_ctx, which, shape, level):
    m, n, k = shape
    x, wg, wu, _ = inputs(np.random.default_rng(m), m, n, k)
    (wg if which == "gate" else wu)[:] *= np.float32(level)
    h, a, u = (Dev(gpu_ctx, np.full((m, n), np.nan, np.float32)) for _ in range(3))
    call(gpu_ctx, "nrs_gated_linear_fwd", Dev(gpu_ctx, x), Dev(gpu_ctx, wg), Dev(gpu_ctx, wu), h, a, u, m, n, k, SILU)
    for got, w in ((a.get(), wg), (u.get(), wu)):
        assert rel_l2(got, x.astype(np.float64) @ w) <= 3 * 8 * U


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_a_gradient_far_below_the_other(gpu_ctx, shape, level):
    """A gate whose weights are small: its pre-activations, and so the other matrix's gradient, are as small."""
    m, n, k = shape
    x, wg, wu, dh = inputs(np.random.default_rng(m), m, n, k)
    a, u = ((x.astype(np.float64) @ w).astype(np.float32) for w in (wg, wu))
    # (dx: both of its terms at the same level, or the gate's alone)
    for scaled in (wg, wg * np.float32(level)):
        b = a * np.float32(level)
        got, want = backward(gpu_ctx, x, scaled, wu, b, u, dh), formulas(x, scaled, wu, dh, b, u)
        for name in got:
            assert rel_l2(got[name], want[name]) <= 3 * 8 * U * 1.2, name


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_closed_gates_leave_the_others_their_bits(gpu_ctx, shape):
    """Gates far to the left pass nothing on, and what they are says nothing about the others' magnitudes."""
    m, n, k = shape
    rng = np.random.default_rng(m)
    x, wg, wu, dh = inputs(rng, m, n, k)
    a, u = ((x.astype(np.float64) @ w).astype(np.float32) for w in (wg, wu))
    shut = rng.random((m, n)) < 0.3
    a[shut] = -1e9
    u[shut] *= np.float32(2.0 ** 60)
    got, want = backward(gpu_ctx, x, wg, wu, a, u, dh), formulas(x, wg, wu, dh, a, u)
    for name in got:
        assert rel_l2(got[name], want[name]) <= 3 * 8 * U * 1.2, name


def test_a_weight_of_zeros(gpu_ctx):
    m, n, k = 200, 96, 128
    x, wg, wu, dh = inputs(np.random.default_rng(9), m, n, k)
    zero = np.zeros_like(wu)
    a = (x.astype(np.float64) @ wg).astype(np.float32)
    got, want = backward(gpu_ctx, x, wg, zero, a, np.zeros_like(a), dh), formulas(x, wg, zero, dh, a, np.zeros_like(a))
    assert (got["dx"] == 0).all() and (got["dwg"] == 0).all()
    assert rel_l2(got["dwu"], want["dwu"]) <= 3 * 8 * U * 1.2


@pytest.mark.parametrize("v", [1e12, 1e20, 1e30])
@pytest.mark.parametrize("kind", [GELU, SILU])
def test_values_far_to_the_right(gpu_ctx, kind, v):
    """Gates of 1e12 and more beside ordinary values in the other matrix; x is the identity."""
    m, n, k = 200, 64, 224
    x, wg, wu = np.eye(m, k, dtype=np.float32), np.full((k, n), v, np.float32), np.ones((k, n), np.float32)
    h = Dev(gpu_ctx, np.full((m, n), np.nan, np.float32))
    call(gpu_ctx, "nrs_gated_linear_fwd", Dev(gpu_ctx, x), Dev(gpu_ctx, wg), Dev(gpu_ctx, wu), h, None, None, m, n, k, kind)
    assert (np.abs(h.get() - float(np.float32(v))) <= 16 * U * v).all()
    a, one, dw = np.full((m, n), v, np.float32), np.ones((m, n), np.float32), [Dev(gpu_ctx, np.full((k, n), np.nan, np.float32)) for _ in range(2)]
    call(gpu_ctx, "nrs_gated_linear_bwd", Dev(gpu_ctx, x), None, None, Dev(gpu_ctx, a), Dev(gpu_ctx, one), Dev(gpu_ctx, one), None, *dw, m, n, k, kind, 0, 0)
    assert (np.abs(dw[0].get()[:m] - 1) <= 16 * U).all() and (np.abs(dw[1].get()[:m] - float(np.float32(v))) <= 16 * U * v).all()


FAR = [-8.0, -20.0, -79.0, -81.0, -86.0, -90.0, -1e4, -1e11, -1e12, -1e20, -1e30, -3.4e38, 30.0, 1e4, 1e12, 1e20, 1e30]


def allowed(want, w, a):
    """The sigmoid's argument carries at most five roundings, each of which the exponential makes |w| times as large, and the
    rest some sixteen; results below f32's normal range (w beyond 87, |a| or its slope in front) may come as zeros."""
    return (6 * min(abs(w), 90.0) + 24) * U * np.abs(want) + (4e-36 if w < 0 else 0.0) + 2.0 ** -20 * U * abs(a) * (w > 0)


@pytest.mark.parametrize("kind", [GELU, SILU])
@pytest.mark.parametrize("v", FAR)
@pytest.mark.parametrize("m", [8, 64])                    # f32, and operands as pairs
def test_slopes_far_from_zero(gpu_ctx, m, v, kind):
    """x is the identity, so the weights' gradients are the gates' own."""
    n = 64
    eye, one, a = np.eye(m, dtype=np.float32), np.ones((m, n), np.float32), np.full((m, n), v, np.float32)
    dw = [Dev(gpu_ctx, np.full((m, n), np.nan, np.float32)) for _ in range(2)]
    call(gpu_ctx, "nrs_gated_linear_bwd", Dev(gpu_ctx, eye), None, None, Dev(gpu_ctx, a), Dev(gpu_ctx, one), Dev(gpu_ctx, one), None, *dw, m, n, m, kind, 0, 0)
    f, d, w = act(np.float32(v), kind)
    da, du = dw[0].get(), dw[1].get()
    assert (np.abs(da - d) <= allowed(d, w, 1.0)).all()
    assert (np.abs(da) <= 1.13).all()                     # what no slope exceeds
    assert (np.abs(du - f) <= allowed(f, w, v)).all()


@pytest.mark.parametrize("kind", [GELU, SILU])
@pytest.mark.parametrize("v", FAR)
@pytest.mark.parametrize("m,k", [(1, 64), (4, 64), (16, 64), (64, 256), (200, 224)])   # every form of the forward pass
def test_values_far_from_zero(gpu_ctx, m, k, v, kind):
    n = 64
    x, wg, wu = np.eye(m, k, dtype=np.float32), np.full((k, n), v, np.float32), np.ones((k, n), np.float32)
    h = Dev(gpu_ctx, np.full((m, n), np.nan, np.float32))
    call(gpu_ctx, "nrs_gated_linear_fwd", Dev(gpu_ctx, x), Dev(gpu_ctx, wg), Dev(gpu_ctx, wu), h, None, None, m, n, k, kind)
    f, _, w = act(np.float32(v), kind)
    # (a pair carries a weight to 2^-22: as an error of w it counts |w| times, as one of the value once)
    assert (np.abs(h.get() - f) <= allowed(f, w, v) + 8 * U * (1 + min(abs(w), 90.0)) * np.abs(f)).all()


@pytest.mark.parametrize("kind", [GELU, SILU])
def test_nan_and_infinite_gates(gpu_ctx, kind):
    m = n = 32
    x, wu = np.eye(m, dtype=np.float32), np.ones((m, n), np.float32)
    wg = np.ones((m, n), np.float32)
    wg[0], wg[1] = np.nan, np.inf
    h = Dev(gpu_ctx, shape=(1, n))
    for row in (0, 1):
        call(gpu_ctx, "nrs_gated_linear_fwd", Dev(gpu_ctx, x[row:row + 1]), Dev(gpu_ctx, wg), Dev(gpu_ctx, wu), h, None, None, 1, n, m, kind)
        assert not np.isfinite(h.get()).any()
    dw = [Dev(gpu_ctx, shape=(m, n)) for _ in range(2)]
    a = np.ones((m, n), np.float32)
    a[3, 5] = np.nan
    call(gpu_ctx, "nrs_gated_linear_bwd", Dev(gpu_ctx, x), None, None, Dev(gpu_ctx, a), Dev(gpu_ctx, wu), Dev(gpu_ctx, wu), None, *dw, m, n, m, kind, 0, 0)
    for t in dw:
        assert np.isnan(t.get()[3, 5])


def test_closed_gates_of_the_lowest_value(gpu_ctx):
    m, n, k = 200, 100, 136
    rng = np.random.default_rng(m)
    x, wg, wu, dh = inputs(rng, m, n, k)
    a, u = ((x.astype(np.float64) @ w).astype(np.float32) for w in (wg, wu))
    a[rng.random((m, n)) < 0.3] = np.finfo(np.float32).min
    got, want = backward(gpu_ctx, x, wg, wu, a, u, dh), formulas(x, wg, wu, dh, a, u)
    for name in got:
        assert rel_l2(got[name], want[name]) <= 3 * 8 * U * 1.2, name


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 4])   # a column a lane, and four
def test_as_many_columns_as_an_int_counts(gpu_ctx, n):
    l, w, h = _lib.lib(), Dev(gpu_ctx, shape=(n,), zero=True), Dev(gpu_ctx, shape=(n,))
    ones, at = np.ones(40, np.float32), lambda d, i: C.c_void_p(d.ptr.value + 4 * i)
    spots = [0, n // 2, n - 40]
    for i in spots:
        _lib.check(gpu_ctx.h, l.nrs_h2d(gpu_ctx.h, at(w, i), C.c_void_p(ones.ctypes.data), ones.nbytes))
    call(gpu_ctx, "nrs_gated_linear_fwd", Dev(gpu_ctx, np.full((1, 1), 2.0, np.float32)), w, w, h, None, None, 1, n, 1, 1)   # relu(2 w) * 2 w
    for i in spots:
        got = np.empty(48, np.float32)
        first = max(0, min(i - 4, n - 48))
        _lib.check(gpu_ctx.h, l.nrs_d2h(gpu_ctx.h, C.c_void_p(got.ctypes.data), at(h, first), got.nbytes))
        inside = (first + np.arange(48) >= i) & (first + np.arange(48) < i + 40)
        assert np.array_equal(got, np.where(inside, 4.0, 0.0).astype(np.float32))
