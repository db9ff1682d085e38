"""GELU and its slope far from zero, where the exponential leaves f32's range: element by element, and in a layer's epilogue."""
import numpy as np
import pytest

from neuralrs_b200.cuda import Node, backward_graph, nn
from neuralrs_b200.cuda import runtime as gpu
from .gpu_util import Dev, call

pytestmark = pytest.mark.gpu
FAR = np.array([-5.0, -9.0, -9.5, -10.0, -11.0, -100.0, -1e11, -1e12, -1e15, -1e20, -1e30, -3.4e38, 0.0, 11.0, 1e4, 1e12, 1e20, 1e30, 3.4e38], np.float32)


def gelu(x):
    x = x.astype(np.float64)
    w = 2 * 0.7978845608 * (x + 0.044715 * x ** 3)
    with np.errstate(over="ignore"):
        s, r = 1 / (1 + np.exp(-w)), 1 / (1 + np.exp(w))
        d = s + np.where(s * r > 0, x * (s * r) * 2 * 0.7978845608 * (1 + 3 * 0.044715 * x * x), 0.0)
    return x * s, d


def close(got, want, x):
    # an argument of up to 90 with six roundings in it, each a relative error of its exponential; what is smaller than that
    # leaves of f32's range may come as zero
    return (np.abs(got - want) <= 90 * 8 * 2.0 ** -24 * np.abs(want) + 4e-36).all()


def test_element_by_element(gpu_ctx):
    f, d = gelu(FAR)
    x, y, dx = Dev(gpu_ctx, FAR), Dev(gpu_ctx, np.full_like(FAR, np.nan)), Dev(gpu_ctx, np.full_like(FAR, np.nan))
    call(gpu_ctx, "nrs_gelu_fwd", x, y, FAR.size)
    call(gpu_ctx, "nrs_gelu_bwd", x, Dev(gpu_ctx, np.ones_like(FAR)), dx, FAR.size, 0)
    assert close(y.get(), f, FAR)
    assert close(dx.get(), d, FAR)
    nan = Dev(gpu_ctx, np.array([np.nan], np.float32))
    call(gpu_ctx, "nrs_gelu_fwd", nan, y, 1)
    call(gpu_ctx, "nrs_gelu_bwd", nan, Dev(gpu_ctx, np.ones(1, np.float32)), dx, 1, 0)
    assert np.isnan(y.get()[0]) and np.isnan(dx.get()[0])


@pytest.mark.parametrize("m", [4, 64])                    # f32, and the tensor cores
def test_in_an_epilogue(gpu_ctx, m):
    """Pre-activations from the bias alone: the weights are zeros."""
    n = FAR.size
    w, b = np.zeros((32, 32), np.float32), np.zeros(32, np.float32)
    b[:n] = FAR
    nodes = [Node.new(v, v.shape) for v in (np.ones((m, 32), np.float32), w, b)]
    for v in nodes:
        gpu.to_cuda(v)
    out = nn.linear_act(*nodes, 2)
    f, d = gelu(FAR)
    assert close(gpu.to_host(out).reshape(m, 32)[:, :n], f, FAR)
    gpu.set_grad(out, np.ones((m, 32), np.float32))
    backward_graph(out)
    got = gpu.read_grad(nodes[2])[:n]
    assert close(got / m, d, FAR)
