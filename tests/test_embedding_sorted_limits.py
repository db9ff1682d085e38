"""The embedding gradient's sizes at the ends of their ranges."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib
from .gpu_util import Dev, call

WIDEST = 2 ** 31 - 1


@pytest.mark.parametrize("dim", [WIDEST - 200, WIDEST - 127, WIDEST - 126, WIDEST])
def test_workspace_of_wide_rows(nrs_lib, dim):
    # two rows of sums for each piece of the tokens, and what the sort leaves
    assert nrs_lib.nrs_embedding_sorted_workspace(10, dim, 10) >= 2 * 4 * dim + 8 * 10 + 4 * 11


@pytest.mark.gpu
def test_the_widest_row(gpu_ctx):
    l, n = _lib.lib(), WIDEST
    need = l.nrs_embedding_sorted_workspace(2, n, 1)
    g, dw, ws = Dev(gpu_ctx, shape=(2 * n,), zero=True), Dev(gpu_ctx, shape=(n,)), Dev(gpu_ctx, shape=(need,), dtype=np.uint8)
    part, at = np.arange(1, 41, dtype=np.float32), lambda d, i: C.c_void_p(d.ptr.value + 4 * i)
    spots = [0, n // 2, n - 40]
    for i in spots:
        for t in (0, n):
            _lib.check(gpu_ctx.h, l.nrs_h2d(gpu_ctx.h, at(g, t + i), C.c_void_p(part.ctypes.data), part.nbytes))
    call(gpu_ctx, "nrs_embedding_sorted_bwd", g, Dev(gpu_ctx, np.zeros(2, np.int32)), dw, 2, n, 1, C.c_float(3.0), 0, ws, need)
    for i in spots:
        got = np.empty(40, np.float32)
        _lib.check(gpu_ctx.h, l.nrs_d2h(gpu_ctx.h, C.c_void_p(got.ctypes.data), at(dw, i), got.nbytes))
        assert np.array_equal(got, 6 * part)
