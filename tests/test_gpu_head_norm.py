"""Norms of query and key heads with the rotation of their positions, against the formulas in 64 bits; the formulas' own
gradient against differences; layouts, strides, positions, captured calls and refusals."""
import ctypes as C

import numpy as np
import pytest

from neuralrs_b200 import _lib, cuda
from neuralrs_b200.cuda import Node, backward_graph, graph, nn
from neuralrs_b200.cuda import runtime as gpu
from .gpu_util import Dev, call

F, U = C.c_float, 2.0 ** -24      # a rounding to f32 is off by at most U of the value
EPS = 1e-6


def angles(positions, rot, base=10000.0):
    a = np.asarray(positions, np.float64)[:, None] * base ** (-np.arange(0, rot, 2) / max(rot, 1))
    return np.cos(a), np.sin(a)


def members(d, rot, inter):
    """Feature indices of the two members of every pair."""
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)


def rotate(z, cs, rot, inter, back=False):
    (c, s), (a, b) = cs, members(z.shape[-1], rot, inter)
    c, s = c[:, None], (-s if back else s)[:, None]
    out = z.copy()
    out[..., a], out[..., b] = z[..., a] * c - z[..., b] * s, z[..., a] * s + z[..., b] * c
    return out


def reach(z, rot, inter):
    """What a pair's members are bounded by: |a| + |b| in place of each."""
    a, b = members(z.shape[-1], rot, inter)
    out = np.abs(z)
    out[..., a] = out[..., b] = out[..., a] + out[..., b]
    return out


def formulas(x, gamma, cs, rot, inter, g=None):
    """x [tokens, heads, d] in 64 bits -> (y, dx, dgamma)."""
    rstd = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    y = rotate(x * rstd * gamma, cs, rot, inter)
    if g is None:
        return y, None, None
    dz = rotate(g, cs, rot, inter, back=True)
    xhat = x * rstd
    dx = rstd * (dz * gamma - xhat * (dz * gamma * xhat).mean(-1, keepdims=True))
    return y, dx, (dz * xhat).sum((0, 1))


@pytest.mark.parametrize("inter", [False, True])
def test_the_formulas_gradient_against_differences(inter):
    rng = np.random.default_rng(0)
    t, h, d, rot = 3, 2, 10, 6
    x, g, gamma = rng.standard_normal((t, h, d)), rng.standard_normal((t, h, d)), 1 + 0.2 * rng.standard_normal(d)
    cs = angles([0, 5, 100000], rot)
    _, dx, dw = formulas(x, gamma, cs, rot, inter, g)
    f = lambda x, gamma: (formulas(x, gamma, cs, rot, inter)[0] * g).sum()
    step = 1e-6
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = step
        assert abs((f(x + e, gamma) - f(x - e, gamma)) / (2 * step) - dx[i]) < 1e-7
    for i in range(d):
        e = np.zeros(d)
        e[i] = step
        assert abs((f(x, gamma + e) - f(x, gamma - e)) / (2 * step) - dw[i]) < 1e-7


def run(ctx, x, gamma, table, positions, seq, rot, inter, g, ld=None, old=None, shift=0):
    """One call each way on [tokens, heads, d] arrays of queries and keys, from rows `ld` floats apart."""
    (xq, xk), (t, hq, d), hk = x, x[0].shape, x[1].shape[1]
    max_len = table.shape[0] if table is not None else 0

    def rows(v, width):                                  # in rows of their own stride, `shift` floats into the buffer
        a = np.full((t, width), 9.0, np.float32)
        a[:, :v.shape[1] * d] = v.reshape(t, -1)
        return Dev(ctx, np.concatenate([np.zeros(shift, np.float32), a.ravel()]))

    at = lambda b: C.c_void_p(b.ptr.value + 4 * shift) if b is not None else None
    ldq, ldk = (ld, ld) if ld else (hq * d, hk * d)
    dev = lambda a: Dev(ctx, a) if a is not None else None
    bq, bk, wq, wk, tab, pos = rows(xq, ldq), rows(xk, ldk), dev(gamma[0]), dev(gamma[1]), dev(table), dev(positions)
    oq, ok = rows(np.zeros_like(xq), ldq), rows(np.zeros_like(xk), ldk)
    shape = (t, seq, hq, hk, d, rot, max_len, int(inter), F(EPS))
    call(ctx, "nrs_qk_norm_rotary_fwd", at(bq), ldq, at(bk), ldk, wq, wk, tab, pos, at(oq), ldq, at(ok), ldk, *shape)
    back = lambda b, h, w: b.get()[shift:].reshape(t, w)
    ys = [back(oq, hq, ldq), back(ok, hk, ldk)]
    for y, h in zip(ys, (hq, hk)):
        assert (y[:, h * d:] == 9.0).all()               # what lies between the rows is left as it was
    ys = [y[:, :h * d].reshape(t, h, d) for y, h in zip(ys, (hq, hk))]
    if g is None:
        return ys
    gq, gk = rows(g[0], ldq), rows(g[1], ldk)
    acc = old is not None
    dq, dk = (rows(old[0], ldq), rows(old[1], ldk)) if acc else (rows(np.zeros_like(xq), ldq), rows(np.zeros_like(xk), ldk))
    dwq, dwk = (Dev(ctx, old[2]), Dev(ctx, old[3])) if acc else (Dev(ctx, shape=(d,)), Dev(ctx, shape=(d,)))
    need = _lib.lib().nrs_qk_norm_rotary_workspace(t, hq, hk, d)
    ws = Dev(ctx, shape=(need,), dtype=np.uint8)
    call(ctx, "nrs_qk_norm_rotary_bwd", at(gq), ldq, at(gk), ldk, at(bq), ldq, at(bk), ldk, wq, wk, tab, pos, at(dq), ldq, at(dk), ldk, dwq, dwk,
         *shape, int(acc), int(acc), ws, need)
    dx = [back(dq, hq, ldq)[:, :hq * d].reshape(t, hq, d), back(dk, hk, ldk)[:, :hk * d].reshape(t, hk, d)]
    return ys, dx, [dwq.get(), dwk.get()]


CASES = [  # tokens, seq, heads_q, heads_k, d, rot, interleaved, positions, stride, shift
    (1, 1, 1, 1, 32, 32, False, None, None, 0),
    (7, 3, 8, 2, 32, 32, False, None, None, 0),
    (130, 128, 4, 4, 64, 32, True, None, 640, 0),
    (33, 33, 5, 3, 128, 128, False, "far", 1200, 0),
    (300, 100, 16, 4, 128, 64, True, "far", None, 0),
    (9, 9, 2, 1, 256, 256, False, None, None, 0),
    (21, 21, 3, 2, 80, 80, False, None, None, 0),       # ten of sixteen lanes
    (21, 21, 3, 2, 96, 48, True, "far", None, 0),
    (40, 40, 2, 1, 8, 8, False, None, None, 0),
    (40, 40, 2, 1, 64, 0, False, None, None, 0),        # norms alone
    (15, 15, 3, 1, 33, 20, False, "far", None, 0),      # from here on: odd sizes, strides and addresses
    (15, 15, 3, 1, 33, 32, True, None, 101, 0),
    (12, 12, 2, 2, 64, 64, False, None, None, 1),
    (12, 12, 2, 2, 64, 20, False, "far", None, 0),
    (5, 5, 2, 1, 2, 2, False, None, None, 0),
    (6, 6, 2, 1, 1, 0, False, None, None, 0),
    (6, 6, 1, 1, 1000, 500, True, None, None, 0),
    (6, 6, 1, 2, 1024, 1024, False, None, None, 0),
    (5000, 77, 3, 1, 64, 64, False, None, None, 0),     # more tasks than warps
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("weights", [True, False])
def test_against_the_formulas(gpu_ctx, case, weights):
    t, seq, hq, hk, d, rot, inter, far, ld, shift = case
    rng = np.random.default_rng(d + t)
    max_len = 200000 if far else max(seq, 1)
    positions = rng.integers(0, max_len, t).astype(np.int32) if far else None
    if far:
        positions[0], positions[-1] = 0, max_len - 1
    at = positions if far else np.arange(t) % seq
    x = [rng.standard_normal((t, h, d)).astype(np.float32) * 1.5 for h in (hq, hk)]
    g = [rng.standard_normal((t, h, d)).astype(np.float32) for h in (hq, hk)]
    x[0][t // 2, 0] = 0.0                                 # a head of zeros: only eps is left
    gamma = [(1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if weights else None for _ in range(2)]
    table = None
    if rot:
        tab = Dev(gpu_ctx, shape=(max_len, rot))
        call(gpu_ctx, "nrs_rotary_table", tab, max_len, rot, F(10000.0))
        table = tab.get()
        c, s = angles(at, rot)
        # the table: one rounding of the 64-bit value, whose angle may be off by a few 2^-53 of itself
        slack = U + 4 * 2.0 ** -53 * max_len
        assert np.abs(table[at, 0::2] - c).max() <= slack and np.abs(table[at, 1::2] - s).max() <= slack
    old = [rng.standard_normal(v.shape).astype(np.float32) for v in (x[0], x[1], np.zeros(d), np.zeros(d))] if weights else None
    ys, dxs, dws = run(gpu_ctx, x, gamma, table, positions, seq, rot, inter, g, ld, old, shift)
    cs = angles(at, rot)
    for i, h in enumerate((hq, hk)):
        x64, g64, w64 = x[i].astype(np.float64), g[i].astype(np.float64), gamma[i].astype(np.float64) if weights else np.ones(d)
        y, dx, dw = formulas(x64, w64, cs, rot, inter, g64)
        # sum of squares: at most 8 + log2(32) or d / 32 + log2(32) additions and a product; half of that in its root, whose
        # function is good to 2 ulp; then 3 products, 2 of the rotation with a rounded cosine, and its sum
        c1 = 0.5 * (15 + d / 32) + 4 + 3 + 3 + 4
        rstd = 1.0 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + EPS)
        assert (np.abs(ys[i] - y) <= c1 * U * reach(x64 * rstd * w64, rot, inter) + 1e-37).all()
        # the gradient: the same for each of its two terms, and a second sum over the head
        dz = reach(g64, rot, inter) * np.abs(w64)
        c2 = 2 * c1 + 15 + d / 32
        bound = c2 * U * rstd * (dz + np.abs(x64 * rstd) * (dz * np.abs(x64 * rstd)).mean(-1, keepdims=True))
        o = old[i].astype(np.float64) if weights else 0.0
        assert (np.abs(dxs[i] - (dx + o)) <= bound + U * np.abs(dx + o) * 1.01 + 1e-37).all()
        terms = t * h
        bound = (c1 + terms + 8) * U * (reach(g64, rot, inter) * np.abs(x64 * rstd)).sum((0, 1))
        o = old[2 + i].astype(np.float64) if weights else 0.0
        assert (np.abs(dws[i] - (dw + o)) <= bound + U * np.abs(dw + o) * 1.01).all()


@pytest.mark.gpu
def test_rotation_keeps_distances(gpu_ctx):
    """The score of a rotated query and key goes by the distance of their positions alone, also far out."""
    d, far = 64, 100000
    rng = np.random.default_rng(3)
    v = rng.standard_normal((1, 1, d)).astype(np.float32)
    tab = Dev(gpu_ctx, shape=(far + 64, d))
    call(gpu_ctx, "nrs_rotary_table", tab, far + 64, d, F(10000.0))
    table = tab.get()
    score = []
    for p in (0, far):
        at = np.array([p + 3, p + 40], np.int32)
        x = np.repeat(v, 2, axis=0)
        q, k = run(gpu_ctx, [x, x], [None, None], table, at, 2, d, False, None)
        score.append(float(q[0, 0].astype(np.float64) @ k[1, 0]))
    # 64 products of values around 1, each off by the 20 roundings or so of the test above
    assert abs(score[0] - score[1]) < 64 * 4 * 20 * U * 4


@pytest.mark.gpu
def test_in_place_and_one_side_alone(gpu_ctx):
    rng = np.random.default_rng(4)
    t, h, d = 50, 4, 64
    x = rng.standard_normal((t, h * d)).astype(np.float32)
    gamma = rng.standard_normal(d).astype(np.float32)
    g = rng.standard_normal((t, h * d)).astype(np.float32)
    w, src, dst = Dev(gpu_ctx, gamma), Dev(gpu_ctx, x), Dev(gpu_ctx, shape=x.shape)
    shape = (t, t, h, 0, d, 0, 0, 0, F(EPS))
    call(gpu_ctx, "nrs_qk_norm_rotary_fwd", src, h * d, None, 0, w, None, None, None, dst, h * d, None, 0, *shape)
    want = dst.get()
    call(gpu_ctx, "nrs_qk_norm_rotary_fwd", src, h * d, None, 0, w, None, None, None, src, h * d, None, 0, *shape)
    assert np.array_equal(src.get(), want)
    need = _lib.lib().nrs_qk_norm_rotary_workspace(t, h, 0, d)
    ws, dg, dx, src = Dev(gpu_ctx, shape=(need,), dtype=np.uint8), Dev(gpu_ctx, g), Dev(gpu_ctx, shape=x.shape), Dev(gpu_ctx, x)
    args = lambda out: (dg, h * d, None, 0, src, h * d, None, 0, w, None, None, None, out, h * d, None, 0, None, None, *shape, 0, 0, ws, need)
    call(gpu_ctx, "nrs_qk_norm_rotary_bwd", *args(dx))
    want = dx.get()
    call(gpu_ctx, "nrs_qk_norm_rotary_bwd", *args(dg))
    assert np.array_equal(dg.get(), want)


@pytest.mark.gpu
def test_positions_outside_the_table_are_reported(gpu_ctx):
    rng = np.random.default_rng(5)
    for d, rot in ((32, 32), (33, 20)):                   # both kernels
        x = [rng.standard_normal((4, 2, d)).astype(np.float32)] * 2
        at = np.array([0, 8, -1, 7], np.int32)
        tab = Dev(gpu_ctx, shape=(8, rot))
        call(gpu_ctx, "nrs_rotary_table", tab, 8, rot, F(10000.0))
        table = tab.get()
        bufs = [Dev(gpu_ctx, x[0].reshape(4, -1)), Dev(gpu_ctx, shape=(4, 2 * d)), Dev(gpu_ctx, table), Dev(gpu_ctx, at)]
        shape = (4, 4, 2, 2, d, rot, 8, 0, F(EPS))
        call(gpu_ctx, "nrs_qk_norm_rotary_fwd", bufs[0], 2 * d, bufs[0], 2 * d, None, None, bufs[2], bufs[3], bufs[1], 2 * d, Dev(gpu_ctx, shape=(4, 2 * d)), 2 * d, *shape)
        with pytest.raises(_lib.NrsError, match="rotation met a position") as e:
            gpu_ctx.sync()
        assert e.value.code == 1
        y = bufs[1].get()
        assert (y[1:3] == 0).all() and (y[0] != 0).any() and (y[3] != 0).any()
        need = _lib.lib().nrs_qk_norm_rotary_workspace(4, 2, 2, d)
        dq, dw = Dev(gpu_ctx, shape=(4, 2 * d)), Dev(gpu_ctx, shape=(d,))
        call(gpu_ctx, "nrs_qk_norm_rotary_bwd", bufs[0], 2 * d, bufs[0], 2 * d, bufs[0], 2 * d, bufs[0], 2 * d, None, None, bufs[2], bufs[3], dq, 2 * d, None, 0,
             dw, None, *shape, 0, 0, Dev(gpu_ctx, shape=(need,), dtype=np.uint8), need)
        with pytest.raises(_lib.NrsError):
            gpu_ctx.sync()
        assert (dq.get()[1:3] == 0).all()
        _, _, want = formulas(x[0][[0, 3]].astype(np.float64), np.ones(d), angles([0, 7], rot), rot, False, x[0][[0, 3]].astype(np.float64))
        assert np.abs(dw.get() - want).max() < 1e-5


@pytest.mark.gpu
def test_captured_calls_replay(gpu_ctx):
    """Forward and backward captured into a graph and replayed on new contents of the same buffers."""
    import torch
    rng = np.random.default_rng(6)
    t, h, d = 64, 4, 32
    s = torch.cuda.Stream()
    ctx = cuda.Context(0)
    ctx.set_stream(s.cuda_stream)
    l = _lib.lib()
    with torch.cuda.stream(s):
        x, g = torch.empty(t, h * d, device="cuda"), torch.empty(t, h * d, device="cuda")
        y, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.empty(d, device="cuda")
        need = l.nrs_qk_norm_rotary_workspace(t, h, 0, d)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        shape = (t, t, h, 0, d, 0, 0, 0, F(EPS))

        def both():
            _lib.check(ctx.h, l.nrs_qk_norm_rotary_fwd(ctx.h, x.data_ptr(), h * d, None, 0, None, None, None, None, y.data_ptr(), h * d, None, 0, *shape))
            _lib.check(ctx.h, l.nrs_qk_norm_rotary_bwd(ctx.h, g.data_ptr(), h * d, None, 0, x.data_ptr(), h * d, None, 0, None, None, None, None, dx.data_ptr(),
                                                       h * d, None, 0, dw.data_ptr(), None, *shape, 0, 0, ws.data_ptr(), need))
        x.normal_()
        g.normal_()
        both()
        s.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            both()
        for _ in range(2):
            x.copy_(torch.from_numpy(rng.standard_normal((t, h * d)).astype(np.float32)))
            g.copy_(torch.from_numpy(rng.standard_normal((t, h * d)).astype(np.float32)))
            gr.replay()
            s.synchronize()
            got = [v.clone() for v in (y, dx, dw)]
            both()
            s.synchronize()
            for a, b in zip(got, (y, dx, dw)):
                assert torch.equal(a, b)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("positions", [False, True])
def test_nodes(gpu_ctx, positions):
    """Through the graph: two results from one call, gradients of both and of the norms' weights."""
    rng = np.random.default_rng(7)
    b, s, hq, hk, d, rot = 2, 9, 4, 2, 32, 16
    q, k = rng.standard_normal((b, s, hq * d)).astype(np.float32), rng.standard_normal((b, s, hk * d)).astype(np.float32)
    wq, wk = (1 + 0.1 * rng.standard_normal(d).astype(np.float32) for _ in range(2))
    gq, gk = rng.standard_normal(q.shape).astype(np.float32), rng.standard_normal(k.shape).astype(np.float32)
    nodes = [Node.new(a, a.shape) for a in (q, k, wq, wk)]
    for n in nodes:
        gpu.to_cuda(n)
    rotary = nn.RotaryEmbedding(rot, 1000)
    at = rng.integers(0, 1000, (b, s)) if positions else None
    norm = nn.HeadNorm(nodes[2], nodes[3], rotary, True, EPS)
    oq, ok = norm.forward(nodes[0], nodes[1], hq, hk, at)
    assert oq.shape == list(q.shape) and ok.shape == list(k.shape)
    cs = angles(at.ravel() if positions else np.arange(b * s) % s, rot)
    for out, x, w, g, h, nx, nw in ((oq, q, wq, gq, hq, nodes[0], nodes[2]), (ok, k, wk, gk, hk, nodes[1], nodes[3])):
        y, dx, dw = formulas(x.reshape(b * s, h, d).astype(np.float64), w.astype(np.float64), cs, rot, True, g.reshape(b * s, h, d).astype(np.float64))
        assert np.abs(gpu.to_host(out) - y.ravel()).max() < 1e-5
        gpu.set_grad(out, g)
        backward_graph(out)
        assert np.abs(gpu.read_grad(nx) - dx.ravel()).max() < 1e-5 * max(1, np.abs(dx).max())
        assert np.abs(gpu.read_grad(nw) - dw).max() < 1e-5 * max(1, np.abs(dw).max())
    for bad in (lambda: norm.forward(nodes[0], nodes[1], hq, hq), lambda: norm.forward(nodes[0], nodes[1], 3, 2),
                lambda: norm.forward(nodes[0], nodes[1], hq, hk, np.full((b, s), 1000)), lambda: norm.forward(nodes[0], nodes[2], hq, hk),
                lambda: nn.HeadNorm(nodes[0], None, rotary).forward(nodes[0], nodes[1], hq, hk)):
        with pytest.raises(_lib.NrsError):
            bad()
    with pytest.raises(_lib.NrsError):
        nn.RotaryEmbedding(7, 10)


@pytest.mark.gpu
def test_refusals(gpu_ctx):
    b = Dev(gpu_ctx, shape=(4, 64), zero=True)
    big = (4, 4, 2, 0, 32, 32, 8, 0, F(EPS))

    def fwd(shape, x=b, out=b, ld=64, table=b, ld_out=64):
        call(gpu_ctx, "nrs_qk_norm_rotary_fwd", x, ld, None, 0, None, None, table, None, out, ld_out, None, 0, *shape)

    for kw, code in [(dict(shape=big, x=None), 1), (dict(shape=big, ld=32), 2), (dict(shape=big, table=None), 1), (dict(shape=big, ld_out=68), 1),
                     (dict(shape=(4, 9, 2, 0, 32, 31, 8, 0, F(EPS))), 2), (dict(shape=(4, 4, 2, 0, 32, 34, 8, 0, F(EPS))), 2),
                     (dict(shape=(9, 9, 2, 0, 32, 32, 8, 0, F(EPS))), 2), (dict(shape=(4, 0, 2, 0, 32, 32, 8, 0, F(EPS))), 2),
                     (dict(shape=(-1, 4, 2, 0, 32, 32, 8, 0, F(EPS))), 2), (dict(shape=(4, 4, 2, 0, 1025, 32, 8, 0, F(EPS))), 7),
                     (dict(shape=(4, 4, 2, 0, 32, 32, 8, 0, F(-1.0))), 1), (dict(shape=(1, 1, 1 << 27, 0, 32, 32, 8, 0, F(EPS))), 2)]:
        with pytest.raises(_lib.NrsError) as e:
            fwd(**kw)
        assert e.value.code == code, kw
    fwd((0, 4, 2, 0, 32, 32, 8, 0, F(EPS)), x=None, out=None)                     # no tokens: nothing to do
    need = _lib.lib().nrs_qk_norm_rotary_workspace(4, 2, 0, 32)
    for ws, nbytes, acc in ((None, need, 0), (b, need - 1, 0), (C.c_void_p(b.ptr.value + 4), need, 0), (b, 1 << 20, 1)):
        with pytest.raises(_lib.NrsError) as e:           # the last: in place and adding
            call(gpu_ctx, "nrs_qk_norm_rotary_bwd", b, 64, None, 0, b, 64, None, 0, None, None, b, None, b, 64, None, 0, None, None, *big, acc, 0, ws, nbytes)
        assert e.value.code == 1
    # no tokens: the weights' gradients are zeros, or stay
    w = Dev(gpu_ctx, np.ones(32, np.float32))
    none = (0, 4, 2, 0, 32, 0, 0, 0, F(EPS))
    call(gpu_ctx, "nrs_qk_norm_rotary_bwd", None, 64, None, 0, None, 64, None, 0, None, None, None, None, None, 64, None, 0, w, None, *none, 0, 1, None, 0)
    assert (w.get() == 1).all()
    call(gpu_ctx, "nrs_qk_norm_rotary_bwd", None, 64, None, 0, None, 64, None, 0, None, None, None, None, None, 64, None, 0, w, None, *none, 0, 0, None, 0)
    assert (w.get() == 0).all()


def test_null_context_is_refused(nrs_lib):
    assert nrs_lib.nrs_rotary_table(None, None, 1, 2, F(1.0)) == 1
    assert nrs_lib.nrs_qk_norm_rotary_workspace(0, 1, 1, 8) == 0
