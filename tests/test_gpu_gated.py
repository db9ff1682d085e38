"""Gated feed-forward layers against the formulas in 64 bits, in every math mode and at sizes around each form's limits; the
formulas' gradient against differences; accumulation, masks of rows, captured calls, nodes and refusals."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib, cuda
from neuralrs_b200.cuda import Node, backward_graph, graph, nn
from neuralrs_b200.cuda import runtime as gpu
from .conftest import rel_l2
from .gpu_util import Dev, call

F, U = C.c_float, 2.0 ** -24
NONE, RELU, GELU, SILU = 0, 1, 2, 3


def act(a, kind):
    if kind == NONE:
        return a, np.ones_like(a)
    if kind == RELU:
        return np.maximum(a, 0), (a > 0).astype(a.dtype)
    if kind == SILU:
        s = 1 / (1 + np.exp(-a))
        return a * s, s * (1 + a * (1 - s))
    v = 0.7978845608 * (a + 0.044715 * a ** 3)
    t = np.tanh(v)
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * 0.7978845608 * (1 + 3 * 0.044715 * a * a)


def formulas(x, wg, wu, kind, dh):
    a, u = x @ wg, x @ wu
    f, d = act(a, kind)
    da, du = dh * u * d, dh * f
    return dict(h=f * u, a=a, u=u, dx=da @ wg.T + du @ wu.T, dwg=x.T @ da, dwu=x.T @ du, da=da, du=du)


@pytest.mark.parametrize("kind", [NONE, RELU, GELU, SILU])
def test_the_formulas_gradient_against_differences(kind):
    rng = np.random.default_rng(0)
    x, wg, wu, dh = rng.standard_normal((3, 4)), rng.standard_normal((4, 5)), rng.standard_normal((4, 5)), rng.standard_normal((3, 5))
    want = formulas(x, wg, wu, kind, dh)
    f = lambda *p: (formulas(*p, kind, dh)["h"] * dh).sum()
    for name, i in (("dx", 0), ("dwg", 1), ("dwu", 2)):
        p = [x, wg, wu]
        for at in np.ndindex(p[i].shape):
            e = np.zeros_like(p[i])
            e[at] = 1e-6
            q = [v + e if j == i else v for j, v in enumerate(p)]
            r = [v - e if j == i else v for j, v in enumerate(p)]
            assert abs((f(*q) - f(*r)) / 2e-6 - want[name][at]) < 1e-7


def inputs(rng, m, n, k):
    s = 1 / np.sqrt(max(k, 1))
    return [v.astype(np.float32) for v in (rng.standard_normal((m, k)), rng.standard_normal((k, n)) * s, rng.standard_normal((k, n)) * s, rng.standard_normal((m, n)))]


def run(ctx, x, wg, wu, dh, kind, old=None, keep=True):
    (m, k), n = x.shape, wg.shape[1]
    dev = [Dev(ctx, v) for v in (x, wg, wu, dh)]
    h, a, u = (Dev(ctx, np.full((m, n), np.nan, np.float32)) for _ in range(3))
    call(ctx, "nrs_gated_linear_fwd", dev[0], dev[1], dev[2], h, a if keep else None, u if keep else None, m, n, k, kind)
    if not keep:
        return dict(h=h.get())
    out = [Dev(ctx, v if old else np.full_like(v, np.nan)) for v in (old or (x, wg, wu))]
    call(ctx, "nrs_gated_linear_bwd", dev[0], dev[1], dev[2], a, u, dev[3], *out, m, n, k, kind, int(bool(old)), int(bool(old)))
    return dict(h=h.get(), a=a.get(), u=u.get(), dx=out[0].get(), dwg=out[1].get(), dwu=out[2].get())


# What a mode may err by in a product, relative to the norm of the absolute products (|x| |w|), whose random sum of k terms is
# some sqrt(k) smaller: f32 and pairs in chains of 256 at most 2^-24 per addition of a chain, tensor cores' truncated sums
# 2^-23 per UMMA of 16 values and chain: 16 a chain, plus a rounding for each chain and the operands' 2^-23 each.
def unit(mode, k):
    if mode == _lib.MATH_FP32:
        return U * (k + 2)
    if mode == _lib.MATH_TF32:
        return 2.0 ** -9 + k * 2.0 ** -23             # (an operand read in place is cut to 11 bits, not rounded)
    return 2.0 ** -23 * (16 + k / 256 + 4) if k >= 32 else U * (k + 2)


SHAPES = [(1, 1, 1), (1, 128, 64), (1, 2752, 1024), (2, 33, 65), (3, 100, 37), (5, 96, 2000), (15, 64, 300), (15, 70, 31), (16, 31, 40), (16, 64, 64), (17, 33, 35),
          (64, 32, 32), (100, 200, 72), (129, 129, 129), (128, 64, 1024), (300, 500, 777), (1000, 96, 64), (257, 1024, 320), (40, 2000, 2000), (2500, 72, 40),
          (5, 2000, 1000), (9, 1000, 1000), (15, 68, 8000), (32, 100, 100), (33, 260, 300), (128, 1000, 260), (127, 68, 500), (100, 64, 2500)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [NONE, RELU, GELU, SILU])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("mode", [_lib.MATH_3XTF32, _lib.MATH_FP32, _lib.MATH_TF32], ids=["3xtf32", "fp32", "tf32"])
def test_against_the_formulas(gpu_ctx, mode, shape, kind):
    m, n, k = shape
    rng = np.random.default_rng(m + n + k)
    x, wg, wu, dh = inputs(rng, m, n, k)
    gpu_ctx.set_math_mode(mode)
    try:
        got = run(gpu_ctx, x, wg, wu, dh, kind)
        alone = run(gpu_ctx, x, wg, wu, dh, kind, keep=False)
        old = [rng.standard_normal(v.shape).astype(np.float32) for v in (x, wg, wu)]
        added = run(gpu_ctx, x, wg, wu, dh, kind, old)
    finally:
        gpu_ctx.set_math_mode(_lib.MATH_3XTF32)
    if kind == RELU:   # what lies within rounding of 0 goes by the device's own sign
        ref = formulas(*(v.astype(np.float64) for v in (x, wg, wu)), kind, dh.astype(np.float64))
        assert (np.abs(ref["a"][(got["a"] > 0) != (ref["a"] > 0)]) < unit(mode, k) * 8 * np.sqrt(k + 1)).all()
        a, u = np.where(got["a"] > 0, np.abs(ref["a"]), -np.abs(ref["a"])), ref["u"]
        f, d = act(a, kind)
        da, du = dh * u * d, dh * f
        want = dict(ref, h=f * u, da=da, du=du, dx=da @ wg.T.astype(np.float64) + du @ wu.T, dwg=x.T.astype(np.float64) @ da, dwu=x.T.astype(np.float64) @ du)
    else:
        want = formulas(*(v.astype(np.float64) for v in (x, wg, wu)), kind, dh.astype(np.float64))
    size = lambda p, q: np.linalg.norm(np.abs(p).astype(np.float64) @ np.abs(q))
    e = unit(mode, k)                                     # projections, relative to the norm of |x| |w|
    proj = {"a": e * size(x, wg), "u": e * size(x, wu)}
    for name in ("a", "u"):
        assert np.linalg.norm(got[name] - want[name]) <= proj[name] + 1e-30
    # h, da, du: the errors of a and u through factors that no value exceeds (act's slope is at most 1.13), and 8 roundings
    # and the exponential's 2 ulp of each
    top = lambda v: np.abs(v).max()
    err_h = 1.13 * proj["a"] * top(want["u"]) + proj["u"] * top(act(want["a"], kind)[0]) + 12 * U * np.linalg.norm(np.abs(want["a"] * want["u"]))
    assert np.linalg.norm(got["h"] - want["h"]) <= err_h + 1e-30
    if mode == _lib.MATH_3XTF32 or k < 32 or m < 16 or n < 32:
        assert np.array_equal(alone["h"], got["h"])       # what is kept changes nothing
    curve = 1.6                                           # |act''|
    err_da = top(dh) * (1.13 * proj["u"] + curve * top(want["u"]) * proj["a"]) + 16 * U * np.linalg.norm(np.abs(dh * want["u"]) * (1 + np.abs(want["a"])))
    err_du = top(dh) * 1.13 * proj["a"] + 12 * U * np.linalg.norm(np.abs(dh * want["a"]))
    en, em = unit(mode, 2 * n), unit(mode, m)
    if m < 16 or n < 32 or k < 32:                        # smaller than the tensor cores take: f32, whatever the length
        en, em = max(en, U * (2 * n + 2)), max(em, U * (m + 2))
    if mode == _lib.MATH_3XTF32:                          # a pair's values far below the largest of their tensor
        en, em = en + 2.0 ** -23, em + 2.0 ** -23
    spec = lambda w: np.linalg.norm(w.astype(np.float64), 2)
    bounds = {"dx": en * (size(want["da"], wg.T) + size(want["du"], wu.T)) + err_da * spec(wg) + err_du * spec(wu),
              "dwg": em * size(x.T, want["da"]) + err_da * spec(x), "dwu": em * size(x.T, want["du"]) + err_du * spec(x)}
    for i, name in enumerate(("dx", "dwg", "dwu")):
        assert np.linalg.norm(got[name] - want[name]) <= bounds[name] + 1e-30, name
        # adding: the sum's rounding besides
        assert np.linalg.norm(added[name] - (got[name].astype(np.float64) + old[i])) <= 2 * bounds[name] + 2 * U * np.linalg.norm(np.abs(old[i]) + np.abs(got[name]))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(512, 512, 1024), (256, 1024, 4096), (4096, 256, 512), (200, 5000, 64)], ids=lambda s: "x".join(map(str, s)))
def test_long_sums_err_like_f32(gpu_ctx, shape):
    """Reductions over thousands of values in the default mode: chains of 256, so the error stays that of f32 sums."""
    m, n, k = shape
    rng = np.random.default_rng(m)
    x, wg, wu, dh = inputs(rng, m, n, k)
    got = run(gpu_ctx, x, wg, wu, dh, SILU)
    want = formulas(*(v.astype(np.float64) for v in (x, wg, wu)), SILU, dh.astype(np.float64))
    for name in ("h", "dx", "dwg", "dwu"):
        # 16 truncated additions of a UMMA's 16 values in a chain: their mean error, 2^-24 of a partial sum each, is some
        # 16/2 of them of the chain's sum; the same for each chain's share; a factor of 3 covers the formula's two stages
        assert rel_l2(got[name], want[name]) <= 3 * 8 * U * 1.2, name


@pytest.mark.gpu
def test_weak_rows_and_empty_rows(gpu_ctx):
    """Rows of zeros (padding), and rows a thousand times weaker than the rest, keep their own relative error."""
    rng = np.random.default_rng(5)
    x, wg, wu, dh = inputs(rng, 200, 192, 256)
    x[::3] = 0
    x[1::3] *= np.float32(2.0 ** -10)
    dh[::3] = 0
    got = run(gpu_ctx, x, wg, wu, dh, SILU)
    want = formulas(*(v.astype(np.float64) for v in (x, wg, wu)), SILU, dh.astype(np.float64))
    assert (got["h"][::3] == 0).all() and (got["dx"][::3] == 0).all()
    for rows in (slice(1, None, 3), slice(2, None, 3)):
        for name in ("h", "a", "u", "dx"):
            assert rel_l2(got[name][rows], want[name][rows]) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 64, 64), (64, 64, 64)])
def test_infinities_stay_in_their_row(gpu_ctx, shape):
    m, n, k = shape
    x, wg, wu, dh = inputs(np.random.default_rng(6), m, n, k)
    x[1, 5], dh[1, 7] = np.inf, np.nan
    with np.errstate(all="ignore"):
        got = run(gpu_ctx, x, wg, wu, dh, SILU)
    assert not np.isfinite(got["h"][1]).all() and not np.isfinite(got["dx"][1]).all()
    rest = np.arange(m) != 1
    want = formulas(*(v.astype(np.float64) for v in (x[rest], wg, wu)), SILU, dh[rest].astype(np.float64))
    for name in ("h", "dx"):
        assert rel_l2(got[name][rest], want[name]) < 1e-5
    assert not np.isfinite(got["dwg"]).all()


# The form that reads the weights as they lie (16 to 32 rows, and to 128 from 256 values of k on; 16, 32, 64 and 128 columns).
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(16, 64, 64), (20, 96, 100), (50, 128, 256), (128, 64, 300)], ids=lambda s: "x".join(map(str, s)))
def test_infinities_stay_in_their_row_of_few(gpu_ctx, shape):
    m, n, k = shape
    x, wg, wu, dh = inputs(np.random.default_rng(7), m, n, k)
    x[1, 5], x[3, 0] = np.inf, np.nan
    with np.errstate(all="ignore"):
        got = run(gpu_ctx, x, wg, wu, dh, SILU, keep=False)["h"]
    assert not np.isfinite(got[1]).all() and not np.isfinite(got[3]).any()
    rest = np.setdiff1d(np.arange(m), [1, 3])
    want = formulas(*(v.astype(np.float64) for v in (x[rest], wg, wu)), SILU, dh[rest].astype(np.float64))
    assert rel_l2(got[rest], want["h"]) < 1e-5
    x[1, 5], x[3, 0] = 1.0, 1.0
    wg[2, 9], wu[2, 9] = np.inf, np.inf                   # a column of the weights
    with np.errstate(all="ignore"):
        got = run(gpu_ctx, x, wg, wu, dh, SILU, keep=False)["h"]
    rest = np.setdiff1d(np.arange(n), [9])
    want = formulas(*(v.astype(np.float64) for v in (x, wg[:, rest], wu[:, rest])), SILU, dh[:, rest].astype(np.float64))
    assert rel_l2(got[:, rest], want["h"]) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("m", [16, 100])
def test_captured_calls_of_few_rows_replay(gpu_ctx, m):
    import torch
    s, l, ctx = torch.cuda.Stream(), _lib.lib(), cuda.Context(0)
    ctx.set_stream(s.cuda_stream)
    n, k = 192, 512
    with torch.cuda.stream(s):
        x, wg, wu, h = (torch.randn(*d, device="cuda") for d in ((m, k), (k, n), (k, n), (m, n)))
        f = lambda: _lib.check(ctx.h, l.nrs_gated_linear_fwd(ctx.h, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), None, None, m, n, k, SILU))
        f()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            f()
        # scratch that grows after the capture leaves the graph its own
        big = torch.randn(m, 4096, device="cuda"), torch.randn(4096, 2000, device="cuda"), torch.empty(m, 2000, device="cuda")
        _lib.check(ctx.h, l.nrs_gated_linear_fwd(ctx.h, big[0].data_ptr(), big[1].data_ptr(), big[1].data_ptr(), big[2].data_ptr(), None, None, m, 2000, 4096, SILU))
        for _ in range(2):
            x.copy_(torch.randn(m, k, device="cuda"))
            h.fill_(float("nan"))
            graph.replay()
            s.synchronize()
            a, u = (x.double() @ w.double() for w in (wg, wu))
            want = torch.nn.functional.silu(a) * u
            assert ((h.double() - want).norm() / want.norm()).item() < 1e-5
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 300])
def test_captured_calls_replay(gpu_ctx, m):
    import torch
    s, l, ctx = torch.cuda.Stream(), _lib.lib(), cuda.Context(0)
    ctx.set_stream(s.cuda_stream)
    n, k = 192, 128
    with torch.cuda.stream(s):
        x, wg, wu, dh = (torch.randn(*d, device="cuda") for d in ((m, k), (k, n), (k, n), (m, n)))
        h, a, u, dx, dwg, dwu = (torch.empty(*d, device="cuda") for d in ((m, n), (m, n), (m, n), (m, k), (k, n), (k, n)))

        def both():
            p = lambda *ts: [t.data_ptr() for t in ts]
            _lib.check(ctx.h, l.nrs_gated_linear_fwd(ctx.h, *p(x, wg, wu, h, a, u), m, n, k, SILU))
            _lib.check(ctx.h, l.nrs_gated_linear_bwd(ctx.h, *p(x, wg, wu, a, u, dh, dx, dwg, dwu), m, n, k, SILU, 0, 0))
        both()
        s.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            both()
        # larger calls make the context's scratch grow; the graph keeps its own
        big = [torch.randn(*d, device="cuda") for d in ((2000, 1024), (1024, 1024), (1024, 1024), (2000, 1024))]
        _lib.check(ctx.h, l.nrs_gated_linear_fwd(ctx.h, *(t.data_ptr() for t in big[:3]), big[3].data_ptr(), None, None, 2000, 1024, 1024, SILU))
        for scale in (1.0, 300.0):
            for t in (x, wg, wu, dh):
                t.normal_().mul_(scale)
            gr.replay()
            s.synchronize()
            got = [t.clone() for t in (h, dx, dwg, dwu)]
            both()
            s.synchronize()
            for p, q in zip(got, (h, dx, dwg, dwu)):
                assert torch.equal(p, q)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6, 40), (2, 50, 40), (3, 7, 33)])
def test_nodes(gpu_ctx, shape):
    rng = np.random.default_rng(8)
    k, n = shape[-1], 64
    m = int(np.prod(shape[:-1]))
    x, wg, wu, dh = inputs(rng, m, n, k)
    want = formulas(*(v.astype(np.float64) for v in (x, wg, wu)), GELU, dh.astype(np.float64))

    def nodes():
        ns = [Node.new(v, s) for v, s in ((x, shape), (wg, [k, n]), (wu, [k, n]))]
        for v in ns:
            gpu.to_cuda(v)
        return ns

    nx, ng, nu = nodes()
    out = nn.gated_linear(nx, ng, nu, GELU)
    assert out.shape == list(shape[:-1]) + [n]
    assert rel_l2(gpu.to_host(out), want["h"]) < 1e-5
    for times in (1, 2):                                  # the second pass adds
        gpu.set_grad(out, dh)
        backward_graph(out)
        for node, name in ((nx, "dx"), (ng, "dwg"), (nu, "dwu")):
            assert rel_l2(gpu.read_grad(node), times * want[name]) < 1e-5
    # one weight that needs no gradient, and one tensor as both
    nx, ng, nu = nodes()
    ng.requires_grad = False
    out = nn.gated_linear(nx, ng, nu, GELU)
    gpu.set_grad(out, dh)
    backward_graph(out)
    assert rel_l2(gpu.read_grad(nu), want["dwu"]) < 1e-5 and (gpu.read_grad(ng) == 0).all()
    nx, ng, _ = nodes()
    both = nn.gated_linear(nx, ng, ng, GELU)
    ref = formulas(x.astype(np.float64), wg.astype(np.float64), wg.astype(np.float64), GELU, dh.astype(np.float64))
    gpu.set_grad(both, dh)
    backward_graph(both)
    assert rel_l2(gpu.read_grad(ng), ref["dwg"] + ref["dwu"]) < 1e-5
    for bad in (lambda: nn.gated_linear(nx, ng, nx, GELU), lambda: nn.gated_linear(nx, ng, ng, 4), lambda: nn.gated_linear(ng, ng, ng, GELU)):
        with pytest.raises(_lib.NrsError):
            bad()


@pytest.mark.gpu
def test_empty_and_refused(gpu_ctx):
    b = Dev(gpu_ctx, np.ones((64, 64), np.float32))
    for args, code in [((b, b, b, None, None, None, 4, 4, 4, SILU), 1), ((None, b, b, b, None, None, 4, 4, 4, SILU), 1), ((b, b, b, b, b, None, 4, 4, 4, SILU), 1),
                       ((b, b, b, b, None, None, -1, 4, 4, SILU), 2), ((b, b, b, b, None, None, 4, 4, 4, 4), 1), ((b, b, b, b, None, None, 4, 4, 4, -1), 1)]:
        with pytest.raises(_lib.NrsError) as e:
            call(gpu_ctx, "nrs_gated_linear_fwd", *args)
        assert e.value.code == code
    for args, code in [((b, b, b, None, b, b, b, b, b, 4, 4, 4, SILU, 0, 0), 1), ((b, b, b, b, b, b, b, b, None, 4, 4, 4, SILU, 0, 0), 1),
                       ((None, b, b, b, b, b, b, b, b, 4, 4, 4, SILU, 0, 0), 1)]:
        with pytest.raises(_lib.NrsError) as e:
            call(gpu_ctx, "nrs_gated_linear_bwd", *args)
        assert e.value.code == code
    with pytest.raises(_lib.NrsError):                    # SiLU belongs to gated layers
        call(gpu_ctx, "nrs_gemm", 0, 0, 4, 4, 4, b, b, b, None, SILU, F(0.0))
    call(gpu_ctx, "nrs_gated_linear_fwd", None, None, None, None, None, None, 0, 4, 4, SILU)
    h, dx, dw = (Dev(gpu_ctx, np.ones((4, 4), np.float32)) for _ in range(3))
    call(gpu_ctx, "nrs_gated_linear_fwd", None, None, None, h, None, None, 4, 4, 0, SILU)      # sums of nothing
    assert (h.get() == 0).all()
    call(gpu_ctx, "nrs_gated_linear_bwd", b, b, b, b, b, b, None, dw, dx, 0, 4, 4, SILU, 0, 1)
    assert (dw.get() == 1).all()
    call(gpu_ctx, "nrs_gated_linear_bwd", b, b, b, b, b, b, None, dw, dx, 0, 4, 4, SILU, 0, 0)
    assert (dw.get() == 0).all() and (dx.get() == 0).all()


def test_null_context_is_refused(nrs_lib):
    assert nrs_lib.nrs_gated_linear_fwd(None, None, None, None, None, None, None, 0, 0, 0, 0) == 1
