"""An attention layer's head norms are among its parameters: listed, updated, and cleared with the others."""
import numpy as np
import pytest

from neuralrs_b200.cuda import Node, backward_graph, nn, optim
from neuralrs_b200.cuda import runtime as gpu


def test_parameters_are_listed():
    a, b = object(), object()
    plain = nn.MultiHeadAttention(1, 2, 3, 4, 64, 4)
    assert plain.parameters() == [1, 2, 3, 4]
    assert nn.MultiHeadAttention(1, 2, 3, 4, 64, 4, head_norm=nn.HeadNorm(a, b)).parameters() == [1, 2, 3, 4, a, b]
    assert nn.MultiHeadAttention(1, 2, 3, 4, 64, 4, head_norm=nn.HeadNorm(None, b)).parameters() == [1, 2, 3, 4, b]
    assert nn.HeadNorm(a, a).parameters() == [a]          # one weight of both sides is one parameter


@pytest.mark.gpu
def test_training_through_the_list(gpu_ctx):
    rng = np.random.default_rng(0)
    d, heads, s = 32, 4, 6
    ws = [Node.new((rng.standard_normal((d, d)) / 6).astype(np.float32), [d, d]) for _ in range(4)]
    gammas = [Node.new(np.ones(d // heads, np.float32), [d // heads]) for _ in range(2)]
    x = Node.new(rng.standard_normal((2, s, d)).astype(np.float32), [2, s, d])
    for n in (*ws, *gammas, x):
        gpu.to_cuda(n)
    mha = nn.MultiHeadAttention(*ws, d, heads, True, nn.HeadNorm(*gammas, nn.RotaryEmbedding(d // heads, s)))
    opt = optim.AdamW(1e-2, 0.9, 0.999, 1e-8, 0.0)
    grads = []
    for _ in range(2):
        out = mha.forward_batch(x)
        gpu.set_grad(out, np.ones((2, s, d), np.float32))
        backward_graph(out)
        grads.append([gpu.read_grad(g) for g in gammas])
        assert all(np.abs(g).max() > 0 for g in grads[-1])
        opt.step(mha.parameters())
        gpu.zero_grad(mha.parameters())
        assert all((gpu.read_grad(p) == 0).all() for p in mha.parameters())
    for g in gammas:
        assert (np.abs(gpu.to_host(g) - 1) > 1e-3).any()
