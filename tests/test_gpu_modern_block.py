"""A transformer block of this day built from its parts, as a user composes it: scaled embedding -> (normed, rotated
attention, residual dropout, LayerNorm) -> (gated feed-forward, residual dropout, LayerNorm) -> cross-entropy, one training
step's loss and every gradient against the same formulas in 64 bits, differentiated by torch."""
import numpy as np
import pytest
import torch

from neuralrs_b200 import _lib, cuda
from neuralrs_b200.cuda import Node, backward_graph, graph, loss, nn, optim
from neuralrs_b200.cuda import runtime as gpu
from .conftest import rel_l2

pytestmark = pytest.mark.gpu
P, EPS, SEED = 0.2, 1e-6, 123


def parameters(rng, vocab, d, heads, ff):
    mk = lambda a, b: (rng.standard_normal((a, b)) / np.sqrt(a)).astype(np.float32)
    dh = d // heads
    around = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    return dict(table=(0.2 * rng.standard_normal((vocab, d))).astype(np.float32), w_q=mk(d, d), w_k=mk(d, d), w_v=mk(d, d), w_o=mk(d, d), gq=around(dh), gk=around(dh),
                n1=around(d), b1=(0.1 * rng.standard_normal(d)).astype(np.float32), n2=around(d), b2=(0.1 * rng.standard_normal(d)).astype(np.float32),
                gate=mk(d, ff), up=mk(d, ff), down=mk(ff, d), head=mk(d, vocab))


def formulas(p, ids, labels, heads, causal, masks):
    """The step in 64 bits -> (loss, gradients)."""
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in p.items()}
    b, s = ids.shape
    vocab, d = p["table"].shape
    dh = d // heads
    x = t["table"][torch.tensor(ids, dtype=torch.long)] * float(np.float32(np.sqrt(d)))
    split = lambda v: v.reshape(b, s, heads, dh).transpose(1, 2)
    rms = lambda v, g: v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * g
    angle = torch.arange(s, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64) / dh)
    c, sn = angle.cos(), angle.sin()

    def turn(v):
        u, w = v[..., :dh // 2], v[..., dh // 2:]
        return torch.cat([u * c - w * sn, u * sn + w * c], -1)

    q, k, v = (split(x @ t[n]) for n in ("w_q", "w_k", "w_v"))
    q, k = turn(rms(q, t["gq"])), turn(rms(k, t["gk"]))
    scores = q @ k.transpose(-1, -2) / np.sqrt(dh)
    if causal:
        scores = scores.masked_fill(torch.triu(torch.ones(s, s, dtype=torch.bool), 1), -1e30)
    a = (torch.softmax(scores, -1) @ v).transpose(1, 2).reshape(b, s, d) @ t["w_o"]
    ln = lambda v, g, o: (v - v.mean(-1, keepdim=True)) / (v.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * g + o
    x1 = ln(x + a * torch.tensor(masks[0]).reshape(b, s, d), t["n1"], t["b1"])
    h = torch.nn.functional.silu(x1 @ t["gate"]) * (x1 @ t["up"])
    x2 = ln(x1 + (h @ t["down"]) * torch.tensor(masks[1]).reshape(b, s, d), t["n2"], t["b2"])
    logits = (x2 @ t["head"]).reshape(b * s, vocab)
    out = torch.nn.functional.cross_entropy(logits, torch.tensor(labels, dtype=torch.long))
    out.backward()
    return float(out.detach()), {k: v.grad.numpy() for k, v in t.items()}


class Block:
    def __init__(self, p, heads, causal, s):
        self.n = {k: Node.new(v, v.shape) for k, v in p.items()}
        for v in self.n.values():
            gpu.to_cuda(v)
        n, (vocab, d) = self.n, p["table"].shape
        self.embedding = nn.Embedding(n["table"], vocab, d, scale=d ** 0.5)
        norm = nn.HeadNorm(n["gq"], n["gk"], nn.RotaryEmbedding(d // heads, s), False, EPS)
        self.attention = nn.MultiHeadAttention(n["w_q"], n["w_k"], n["w_v"], n["w_o"], d, heads, causal, norm)
        self.norm1, self.norm2 = nn.LayerNorm(n["n1"], n["b1"]), nn.LayerNorm(n["n2"], n["b2"])

    def forward(self, ids):
        n = self.n
        x = self.embedding.forward_batch(ids)
        b, s, d = x.shape
        x1 = self.norm1.forward(nn.dropout_add(self.attention.forward_batch(x), x, P, True))
        h = nn.gated_linear(graph.reshape(x1, [b * s, d]), n["gate"], n["up"], _lib.ACT_SILU)
        y = graph.reshape(graph.matmul(h, n["down"]), [b, s, d])
        x2 = self.norm2.forward(nn.dropout_add(y, x1, P, True))
        return graph.matmul(graph.reshape(x2, [b * s, d]), n["head"])


@pytest.mark.parametrize("mode", [_lib.MATH_3XTF32, _lib.MATH_FP32], ids=["3xtf32", "fp32"])
@pytest.mark.parametrize("b,s,vocab,d,heads,ff,causal", [(2, 24, 100, 64, 4, 160, True), (1, 1, 50, 32, 2, 48, False), (3, 130, 1000, 128, 4, 344, True)])
def test_training_step(gpu_ctx, oracle32, mode, b, s, vocab, d, heads, ff, causal):
    rng = np.random.default_rng(s)
    p = parameters(rng, vocab, d, heads, ff)
    ids, labels = rng.integers(0, vocab, (b, s)), rng.integers(0, vocab, b * s)
    n = b * s * d
    masks = [oracle32.dropout_mask(n, P, SEED, i * ((n + 3) // 4)).astype(np.float64) for i in range(2)]
    want, grads = formulas(p, ids, labels, heads, causal, masks)
    onehot = np.eye(vocab, dtype=np.float32)[labels]
    gpu_ctx.set_math_mode(mode)
    try:
        block = Block(p, heads, causal, s)
        target = Node.new(onehot, onehot.shape)
        gpu.to_cuda(target)
        _lib.check(gpu_ctx.h, _lib.lib().nrs_rng_seed(gpu_ctx.h, SEED))
        logits = block.forward(ids)
        got = loss.cross_entropy(logits, target)
        loss.cross_entropy_backward(logits, target)
        backward_graph(logits)
        read = {k: gpu.read_grad(v) for k, v in block.n.items()}
        before = {k: gpu.to_host(v) for k, v in block.n.items()}
        opt = optim.AdamW(1e-3, 0.9, 0.999, 1e-8, 0.0)
        opt.step(list(block.n.values()))
        after = {k: gpu.to_host(v) for k, v in block.n.items()}
    finally:
        gpu_ctx.set_math_mode(_lib.MATH_3XTF32)
    # the bar that the framework holds whole models to
    assert abs(got - want) <= 1e-4 * max(1.0, abs(want))
    for k, g in grads.items():
        assert rel_l2(read[k], g) <= 1e-4 or np.linalg.norm(g) < 1e-12, k
    for k in grads:
        moved = np.abs(after[k] - before[k])
        assert moved.max() <= 1.001e-3 + 2e-7 and (np.abs(read[k]).max() == 0 or moved.max() > 0), k


def test_an_eager_graph_lives_while_a_pass_is_captured(gpu_ctx):
    """Nodes of an eager pass stay usable when the same operators are captured on a context of their own and replayed."""
    rng = np.random.default_rng(1)
    p = parameters(rng, 60, 32, 2, 64)
    ids = rng.integers(0, 60, (2, 8))
    block = Block(p, 2, True, 8)
    eager = block.forward(ids)
    seed = rng.standard_normal((16, 60)).astype(np.float32)
    l, s = _lib.lib(), torch.cuda.Stream()
    ctx = cuda.Context(0)
    ctx.set_stream(s.cuda_stream)
    with torch.cuda.stream(s):
        x = torch.randn(64, 32, device="cuda")
        w, h, a, u, dx, dw, du = torch.randn(32, 64, device="cuda"), *(torch.empty(64, 64, device="cuda") for _ in range(3)), torch.empty_like(x), *(torch.empty(32, 64, device="cuda") for _ in range(2))

        def both():
            _lib.check(ctx.h, l.nrs_gated_linear_fwd(ctx.h, x.data_ptr(), w.data_ptr(), w.data_ptr(), h.data_ptr(), a.data_ptr(), u.data_ptr(), 64, 64, 32, 3))
            _lib.check(ctx.h, l.nrs_gated_linear_bwd(ctx.h, x.data_ptr(), w.data_ptr(), w.data_ptr(), a.data_ptr(), u.data_ptr(), h.data_ptr(), dx.data_ptr(),
                                                     dw.data_ptr(), du.data_ptr(), 64, 64, 32, 3, 0, 0))
        both()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            both()
        g.replay()
        s.synchronize()
    gpu.set_grad(eager, seed)
    backward_graph(eager)
    assert all(np.isfinite(gpu.read_grad(v)).all() for v in block.n.values())
    ctx.close()
