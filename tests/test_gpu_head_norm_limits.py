"""Head norms at the limits of what they are given."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib
from .gpu_util import Dev, call

pytestmark = pytest.mark.gpu
F = C.c_float


def backward(ctx, x, g, gamma, eps, table=None, positions=None, old=None, outside=False):
    t, h, d = x.shape
    rot, max_len = (table.shape[1], table.shape[0]) if table is not None else (0, 0)
    need = _lib.lib().nrs_qk_norm_rotary_workspace(t, h, 0, d)
    dx, dw = Dev(ctx, np.full((t, h, d), np.nan, np.float32) if old is None else old), Dev(ctx, np.full(d, np.nan, np.float32))
    call(ctx, "nrs_qk_norm_rotary_bwd", Dev(ctx, g), h * d, None, 0, Dev(ctx, x), h * d, None, 0, Dev(ctx, gamma), None, Dev(ctx, table) if table is not None else None,
         Dev(ctx, positions) if positions is not None else None, dx, h * d, None, 0, dw, None, t, t, h, 0, d, rot, max_len, 0, F(eps), int(old is not None), 0,
         Dev(ctx, shape=(need,), dtype=np.uint8), need)
    if outside:
        with pytest.raises(_lib.NrsError, match="rotation met a position"):
            ctx.sync()
    return dx.get(), dw.get()


def formulas(x, g, gamma, eps):
    x, g, gamma = (v.astype(np.float64) for v in (x, g, gamma))
    rstd = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xhat = x * rstd
    return rstd * (g * gamma - xhat * (g * gamma * xhat).mean(-1, keepdims=True)), (g * xhat).sum((0, 1))


# (16 to 128 rows of these widths fill a block; 33 features take the form for any size)
@pytest.mark.parametrize("t,h,d", [(1, 1, 32), (3, 1, 32), (5, 3, 64), (7, 1, 256), (129, 1, 8), (37, 3, 128), (5, 3, 33)])
def test_no_eps(gpu_ctx, t, h, d):
    rng = np.random.default_rng(t)
    x, g = (rng.standard_normal((t, h, d)).astype(np.float32) for _ in range(2))
    gamma = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    dx, dw = backward(gpu_ctx, x, g, gamma, 0.0)
    want_x, want_w = formulas(x, g, gamma, 0.0)
    assert np.abs(dx - want_x).max() <= 1e-5 * np.abs(want_x).max()
    # the terms' own roundings (some 25 a term) and the sum's
    assert (np.abs(dw - want_w) <= (25 + t * h) * 2.0 ** -24 * (np.abs(g * x).sum((0, 1)) / np.sqrt((x * x).mean(-1)).min())).all()


@pytest.mark.parametrize("d,rot", [(32, 32), (64, 8), (33, 20)])
@pytest.mark.parametrize("add", [False, True])
def test_rows_outside_the_table_hold_anything(gpu_ctx, d, rot, add):
    """Their gradients are zeros whatever they hold, and the weights' gradients do not know them."""
    rng = np.random.default_rng(d)
    t, h = 6, 2
    x, g, old = (rng.standard_normal((t, h, d)).astype(np.float32) for _ in range(3))
    gamma, angle = np.ones(d, np.float32), rng.standard_normal((8, rot // 2))
    table = np.stack([np.cos(angle), np.sin(angle)], -1).reshape(8, rot).astype(np.float32)
    at = np.array([0, 8, 3, -1, 7, 1 << 30], np.int32)
    out = np.array([1, 3, 5])
    x[1], x[3], x[5], g[3], g[5] = np.nan, np.inf, 1e30, np.nan, np.inf
    dx, dw = backward(gpu_ctx, x, g, gamma, 1e-6, table, at, old if add else None, outside=True)
    assert np.array_equal(dx[out], old[out]) if add else (dx[out] == 0).all()
    inside = np.array([0, 2, 4])
    want = backward(gpu_ctx, x[inside], g[inside], gamma, 1e-6, table, at[inside], old[inside] if add else None)
    assert np.abs(dx[inside] - want[0]).max() <= 1e-6 * np.abs(want[0]).max()
    # (the same six terms of a feature, in another order)
    assert (np.abs(dw - want[1]) <= 8 * 2.0 ** -24 * 6 * np.abs(g[inside]).max() * np.abs(x[inside]).max() * 4).all()
