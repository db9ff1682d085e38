"""Embedding lookup with a scale and the table's gradient from sorted tokens, against sums in 64 bits: lengths from one
token to many, runs that cross blocks, ids outside the vocabulary, odd widths and addresses, captured calls, the node and
the trainer's layer."""
import ctypes as C
import pathlib
import subprocess
import sys

import numpy as np
import pytest

from neuralrs_b200 import _lib, cuda, workloads
from neuralrs_b200.cuda import Node, backward_graph, graph, loss, nn
from neuralrs_b200.cuda import runtime as gpu
from .gpu_util import Dev, call

pytestmark = pytest.mark.gpu
F, U = C.c_float, 2.0 ** -24


def ids_of(kind, rng, tokens, vocab):
    if kind == "uniform":
        return rng.integers(0, vocab, tokens)
    if kind == "one":                                    # a padded batch: the same id everywhere
        return np.full(tokens, vocab - 1)
    if kind == "words":                                  # few ids very often
        return np.minimum((rng.pareto(0.6, tokens) * 3).astype(np.int64), vocab - 1)[rng.permutation(tokens)]
    if kind == "outside":
        return rng.integers(-vocab, 2 * vocab, tokens)
    if kind == "descending":
        return (vocab - 1) - np.arange(tokens) * vocab // max(tokens, 1)
    raise ValueError(kind)


def backward(ctx, g, ids, vocab, scale, old=None, shift=0):
    t, d = g.shape
    pad = np.zeros(shift, np.float32)
    dg, di = Dev(ctx, np.concatenate([pad, g.ravel()])), Dev(ctx, ids.astype(np.int32)) if t else None
    dw = Dev(ctx, np.concatenate([pad, (old if old is not None else np.full((vocab, d), np.nan, np.float32)).ravel()]))
    need = _lib.lib().nrs_embedding_sorted_workspace(t, d, vocab)
    guard = 64
    ws = Dev(ctx, np.full(need + guard, 0xAB, np.uint8))  # stale contents must not matter
    at = lambda b: C.c_void_p(b.ptr.value + 4 * shift)
    call(ctx, "nrs_embedding_sorted_bwd", at(dg), di, at(dw), t, d, vocab, F(scale), int(old is not None), ws, need)
    assert (ws.get()[need:] == 0xAB).all()
    return dw.get()[shift:].reshape(vocab, d)


CASES = [  # kind, tokens, dim, vocab, shift
    ("uniform", 1, 4, 1, 0), ("uniform", 1, 256, 1000, 0), ("uniform", 5, 37, 3, 0), ("uniform", 4096, 256, 1000, 0), ("uniform", 4097, 64, 50000, 0),
    ("one", 31, 128, 7, 0), ("one", 32, 128, 1, 0), ("one", 33, 128, 7, 0), ("one", 1000, 256, 300, 0), ("one", 20000, 132, 2000, 0),
    ("words", 300, 8, 40, 0), ("words", 5000, 512, 3000, 0), ("words", 9001, 1024, 70000, 0), ("words", 70001, 4, 11, 0),
    ("outside", 3000, 256, 500, 0), ("outside", 33, 5, 2, 0), ("descending", 8192, 128, 8192, 0), ("descending", 2000, 260, 100000, 0),
    ("uniform", 2000, 99, 333, 0), ("words", 3000, 256, 333, 1), ("words", 129, 1, 9, 0), ("uniform", 16, 3000, 5, 0), ("uniform", 600, 8, 1_300_000, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_gradient(gpu_ctx, case):
    kind, t, d, vocab, shift = case
    rng = np.random.default_rng(t + d)
    ids, scale = ids_of(kind, rng, t, vocab), 3.7
    g = rng.standard_normal((t, d)).astype(np.float32)
    known = (ids >= 0) & (ids < vocab)
    want, size, terms = np.zeros((vocab, d)), np.zeros((vocab, d)), np.zeros(vocab)
    np.add.at(want, ids[known], g[known].astype(np.float64))
    np.add.at(size, ids[known], np.abs(g[known]).astype(np.float64))
    np.add.at(terms, ids[known], 1)
    s = float(np.float32(scale))
    got = backward(gpu_ctx, g, ids, vocab, scale, shift=shift)
    # any order of n - 1 additions is off by at most n - 1 roundings of what is added; then the scale's
    bound = (terms[:, None] + 1) * U * size * s * 1.001
    assert (np.abs(got - want * s) <= bound).all()
    assert (got[terms == 0] == 0).all()
    assert np.array_equal(backward(gpu_ctx, g, ids, vocab, scale, shift=shift), got)      # one order of additions
    old = rng.standard_normal((vocab, d)).astype(np.float32)
    got = backward(gpu_ctx, g, ids, vocab, scale, old, shift)
    assert (np.abs(got - (want * s + old)) <= bound + U * 1.001 * np.abs(want * s + old)).all()
    assert np.array_equal(got[terms == 0], old[terms == 0])


# A block's counts are 128 bytes a row of its share of the vocabulary: on 148 SMs they pass 48 KB, beyond which a launch has to
# ask for its shared memory, in this range.  Each in a process of its own: one larger table asks for all that follow.
@pytest.mark.parametrize("vocab", [56536, 56537, 56700, 56832, 56833])
def test_vocabularies_around_the_default_shared_memory(vocab):
    code = f"""
import ctypes as C
import numpy as np
from neuralrs_b200 import cuda
from tests.test_gpu_embedding_sorted import backward
rng = np.random.default_rng({vocab})
ids, g = rng.integers(0, {vocab}, 500), rng.standard_normal((500, 8)).astype(np.float32)
want = np.zeros(({vocab}, 8))
np.add.at(want, ids, g.astype(np.float64))
got = backward(cuda.Context(0), g, ids, {vocab}, 1.0)
assert np.abs(got - want).max() < 1e-5       # (a few values below 5 a row, each addition off by 2^-24 of them)
assert (got[np.setdiff1d(np.arange({vocab}), ids)] == 0).all()
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=pathlib.Path(__file__).parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_no_tokens(gpu_ctx):
    g, ids = np.zeros((0, 8), np.float32), np.zeros(0, np.int32)
    assert (backward(gpu_ctx, g, ids, 100, 2.0) == 0).all()
    old = np.ones((100, 8), np.float32)
    assert (backward(gpu_ctx, g, ids, 100, 2.0, old) == 1).all()


@pytest.mark.parametrize("t,seq,d,vocab,shift", [(1, 1, 4, 3, 0), (9, 9, 999, 50, 0), (300, 128, 256, 1000, 0), (4096, 128, 64, 1000, 0), (77, 10, 12, 40, 1), (40000, 40000, 36, 7, 0)])
@pytest.mark.parametrize("positions", [False, True])
def test_lookup(gpu_ctx, t, seq, d, vocab, shift, positions):
    rng = np.random.default_rng(t)
    pad = np.zeros(shift, np.float32)
    w, pos = rng.standard_normal((vocab, d)).astype(np.float32), rng.standard_normal((seq, d)).astype(np.float32)
    ids = rng.integers(0, vocab, t).astype(np.int32)
    scale = np.float32(np.sqrt(d))
    dw, dp, out = Dev(gpu_ctx, np.concatenate([pad, w.ravel()])), Dev(gpu_ctx, np.concatenate([pad, pos.ravel()])), Dev(gpu_ctx, shape=(t * d + shift,), zero=True)
    at = lambda b: C.c_void_p(b.ptr.value + 4 * shift)
    call(gpu_ctx, "nrs_embedding_scaled_fwd", at(dw), Dev(gpu_ctx, ids), at(dp) if positions else None, at(out), t, seq if positions else 0, d, vocab, F(scale))
    got = out.get()[shift:].reshape(t, d)
    if not positions:
        assert np.array_equal(got, w[ids] * scale)
    else:
        want = w[ids].astype(np.float64) * float(scale) + pos[np.arange(t) % seq]
        assert (np.abs(got - want) <= U * 1.001 * np.abs(want)).all()                     # one rounding


def test_ids_outside_the_vocabulary(gpu_ctx):
    w, out = Dev(gpu_ctx, np.ones((4, 8), np.float32)), Dev(gpu_ctx, shape=(3, 8))
    call(gpu_ctx, "nrs_embedding_scaled_fwd", w, Dev(gpu_ctx, np.array([0, 4, -1], np.int32)), None, out, 3, 0, 8, 4, F(2.0))
    with pytest.raises(_lib.NrsError, match="outside the vocabulary"):
        gpu_ctx.sync()
    got = out.get()
    assert (got[0] == 2).all() and (got[1:] == 0).all()


def test_captured_calls_replay(gpu_ctx):
    """Two graphs of the same context, each with its workspace, replayed on new ids."""
    import torch
    s, l, ctx = torch.cuda.Stream(), _lib.lib(), cuda.Context(0)
    ctx.set_stream(s.cuda_stream)
    with torch.cuda.stream(s):
        sets = []
        for t, d, vocab in ((700, 64, 90), (3000, 128, 20000)):
            g, ids, dw = torch.randn(t, d, device="cuda"), torch.randint(0, vocab, (t,), device="cuda", dtype=torch.int32), torch.empty(vocab, d, device="cuda")
            need = l.nrs_embedding_sorted_workspace(t, d, vocab)
            ws = torch.empty(need, dtype=torch.uint8, device="cuda")
            run = lambda a=(g, ids, dw, t, d, vocab, ws, need): _lib.check(ctx.h, l.nrs_embedding_sorted_bwd(
                ctx.h, a[0].data_ptr(), a[1].data_ptr(), a[2].data_ptr(), a[3], a[4], a[5], 1.0, 0, a[6].data_ptr(), a[7]))
            run()
            s.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                run()
            sets.append((g, ids, dw, gr))
        for _ in range(3):
            for g, ids, dw, _gr in sets:
                ids.random_(0, dw.shape[0])
                dw.fill_(float("nan"))
            for *_, gr in sets:
                gr.replay()
            s.synchronize()
            for g, ids, dw, _gr in sets:
                want = torch.zeros_like(dw, dtype=torch.float64).index_add_(0, ids.long(), g.double())
                assert float((dw - want).abs().max()) < 1e-4
    ctx.close()


def test_node(gpu_ctx):
    rng = np.random.default_rng(2)
    vocab, d, b, s = 60, 24, 3, 11
    w, ids = rng.standard_normal((vocab, d)).astype(np.float32), rng.integers(0, vocab, (b, s))
    nw = Node.new(w, [vocab, d])
    gpu.to_cuda(nw)
    emb = nn.Embedding(nw, vocab, d, scale=d ** 0.5)
    out = emb.forward_batch(ids)
    assert out.shape == [b, s, d]
    assert np.array_equal(gpu.to_host(out).reshape(b, s, d), w[ids] * np.float32(d ** 0.5))
    one = emb.forward(ids[0])
    assert one.shape == [s, d]
    g = rng.standard_normal((b, s, d)).astype(np.float32)
    gpu.set_grad(out, g)
    gpu.set_grad(one, g[0])
    want = np.zeros((vocab, d))
    np.add.at(want, ids.ravel(), g.reshape(-1, d).astype(np.float64))
    np.add.at(want, ids[0], g[0].astype(np.float64))
    backward_graph(out)
    backward_graph(one)                                   # adds to the first
    assert np.abs(gpu.read_grad(nw).reshape(vocab, d) - want * d ** 0.5).max() < 1e-4
    with pytest.raises(_lib.NrsError, match="out of vocab range"):
        emb.forward([vocab])
    with pytest.raises(_lib.NrsError):
        nn.Embedding(nw, vocab, d, scale=0.0).forward_batch(ids)


def test_trainer_layer(gpu_ctx):
    """A token model whose embedding is scaled equals the unscaled one on a table that already carries the factor (a power of
    two, so both are the same in every bit of the lookup), its table's gradient times the factor."""
    vocab, d, s, b = 50, 16, 12, 4
    rng = np.random.default_rng(3)
    ids, labels = rng.integers(0, vocab, (b, s)).astype(np.int32), rng.integers(0, vocab, b * s).astype(np.int32)
    out = []
    for scaled in (False, True):
        layers = [("embedding", vocab, d, s, int(scaled)), ("transformer_block", d, 2, 32, workloads.ACT_GELU, 1), ("linear", d, vocab)]
        tr = cuda.Trainer(layers, (s,), vocab, ctx=gpu_ctx)
        params = workloads.he_init(layers, 5)
        if not scaled:
            params[0] = params[0] * np.float32(4.0)       # sqrt(16)
        tr.set_params(params)
        l = tr.forward_backward_tokens(ids, labels)
        out.append((l, [tr.get_grad(i) for i in range(tr.n_params)]))
        tr.close()
    (l0, g0), (l1, g1) = out
    assert l0 == l1
    # 48 tokens: either form's sums are off by at most as many roundings of what they add
    assert np.abs(g1[0] - 4 * g0[0]).max() <= 2 * 48 * U * 4 * 48 * np.abs(g0[0]).max()
    for a, c in zip(g0[1:], g1[1:]):
        assert np.array_equal(a, c)


def test_refusals(gpu_ctx):
    b, ids = Dev(gpu_ctx, shape=(1 << 14,), zero=True), Dev(gpu_ctx, np.zeros(8, np.int32))
    need = _lib.lib().nrs_embedding_sorted_workspace(8, 4, 10)
    ok = dict(g=b, idx=ids, dw=b, t=8, d=4, v=10, ws=b, n=need)
    for change, code in [(dict(g=None), 1), (dict(idx=None), 1), (dict(dw=None), 1), (dict(ws=None), 1), (dict(n=need - 1), 1), (dict(t=-1), 2), (dict(d=0), 2),
                         (dict(v=0), 2), (dict(ws=C.c_void_p(b.ptr.value + 4)), 1), (dict(t=(1 << 30) + 1), 2), (dict(v=(1 << 30) + 1), 2)]:
        a = {**ok, **change}
        with pytest.raises(_lib.NrsError) as e:
            call(gpu_ctx, "nrs_embedding_sorted_bwd", a["g"], a["idx"], a["dw"], a["t"], a["d"], a["v"], F(1.0), 0, a["ws"], a["n"])
        assert e.value.code == code, change
    for args, code in [((None, ids, None, b, 8, 0, 4, 10, F(1.0)), 1), ((b, None, None, b, 8, 0, 4, 10, F(1.0)), 1), ((b, ids, b, b, 8, 0, 4, 10, F(1.0)), 2),
                       ((b, ids, None, b, 8, 0, -4, 10, F(1.0)), 2)]:
        with pytest.raises(_lib.NrsError) as e:
            call(gpu_ctx, "nrs_embedding_scaled_fwd", *args)
        assert e.value.code == code
