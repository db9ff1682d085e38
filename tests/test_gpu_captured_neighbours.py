"""Calls beside captures that are not theirs, and graphs beside passes that are not captured."""
import ctypes as C
import glob
import os

import numpy as np
import pytest
import torch

from neuralrs_b200 import _lib, cuda

pytestmark = pytest.mark.gpu
SILU = 3


def cudart():
    import nvidia.cuda_runtime as p
    return C.CDLL(glob.glob(os.path.join(list(p.__path__)[0], "lib", "libcudart.so.*"))[0])


def test_a_call_on_the_legacy_stream_beside_a_capture(gpu_ctx):
    """While a blocking stream is captured, the legacy stream may not even be asked: the call is refused before it launches
    anything, the capture goes on, and afterwards both work."""
    rt, l, ctx = cudart(), _lib.lib(), cuda.Context(0)
    ctx.set_stream(1)                                     # the legacy stream
    m, n, k = 64, 128, 256
    x, wg, wu, h = (torch.randn(*s, device="cuda") for s in ((m, k), (k, n), (k, n), (m, n)))
    torch.cuda.synchronize()
    run = lambda: l.nrs_gated_linear_fwd(ctx.h, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), None, None, m, n, k, SILU)
    assert run() == 0
    torch.cuda.synchronize()
    want = h.clone()
    torch.cuda.synchronize()
    s, g, st = C.c_void_p(), C.c_void_p(), C.c_int(-1)
    assert rt.cudaStreamCreate(C.byref(s)) == 0
    assert rt.cudaStreamBeginCapture(s, 2) == 0           # (relaxed)
    refused = run()
    assert rt.cudaStreamIsCapturing(s, C.byref(st)) == 0
    ended = rt.cudaStreamEndCapture(s, C.byref(g))
    rt.cudaGetLastError()
    if g.value:
        rt.cudaGraphDestroy(g)
    rt.cudaStreamDestroy(s)
    assert refused == 4 and st.value == 1 and ended == 0
    h.zero_()
    torch.cuda.synchronize()
    assert run() == 0
    torch.cuda.synchronize()
    assert torch.equal(h, want)
    ctx.close()


def test_gradients_and_replays_beside_a_capture(gpu_ctx, oracle32):
    """An eager block's gradients are, bit for bit, those of the same block with nothing captured between its passes; and the
    replayed calls leave what the same calls leave eagerly, on other inputs too."""
    from neuralrs_b200.cuda import backward_graph
    from neuralrs_b200.cuda import runtime as gpu
    from .test_gpu_modern_block import Block, formulas, parameters, P, SEED
    rng = np.random.default_rng(1)
    p = parameters(rng, 60, 32, 2, 64)
    ids, labels = rng.integers(0, 60, (2, 8)), rng.integers(0, 60, 16)
    l, ctx, s = _lib.lib(), cuda.Context(0), torch.cuda.Stream()
    ctx.set_stream(s.cuda_stream)

    def captured():
        with torch.cuda.stream(s):
            x, dh = torch.randn(64, 32, device="cuda"), torch.randn(64, 64, device="cuda")
            wg, wu = torch.randn(32, 64, device="cuda"), torch.randn(32, 64, device="cuda")
            h, a, u = (torch.empty(64, 64, device="cuda") for _ in range(3))
            dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)

            def both():
                q = lambda *ts: [t.data_ptr() for t in ts]
                _lib.check(ctx.h, l.nrs_gated_linear_fwd(ctx.h, *q(x, wg, wu, h, a, u), 64, 64, 32, SILU))
                _lib.check(ctx.h, l.nrs_gated_linear_bwd(ctx.h, *q(x, wg, wu, a, u, dh, dx, dwg, dwu), 64, 64, 32, SILU, 0, 0))
            both()
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                both()
            for scale in (1.0, 30.0):
                for t in (x, wg, wu, dh):
                    t.normal_().mul_(scale)
                for t in (h, a, u, dx, dwg, dwu):
                    t.fill_(float("nan"))
                g.replay()
                s.synchronize()
                got = [t.clone() for t in (h, a, u, dx, dwg, dwu)]
                both()
                s.synchronize()
                for t, want in zip(got, (h, a, u, dx, dwg, dwu)):
                    assert torch.equal(t, want)
                pre = [x.double() @ w.double() for w in (wg, wu)]
                want = torch.nn.functional.silu(pre[0]) * pre[1]
                assert float((got[0] - want).norm() / want.norm()) < 1e-5
        return g

    def step(between):
        _lib.check(gpu_ctx.h, l.nrs_rng_seed(gpu_ctx.h, SEED))
        block = Block(p, 2, True, 8)
        logits = block.forward(ids)
        kept = between()
        z = gpu.to_host(logits).reshape(16, 60).astype(np.float64)
        e = np.exp(z - z.max(1, keepdims=True))
        gpu.set_grad(logits, ((e / e.sum(1, keepdims=True) - np.eye(60)[labels]) / 16).astype(np.float32))
        backward_graph(logits)
        del kept
        return {k: gpu.read_grad(v) for k, v in block.n.items()}

    alone, beside = step(lambda: None), step(captured)
    n = 2 * 8 * 32
    masks = [oracle32.dropout_mask(n, P, SEED, i * ((n + 3) // 4)).astype(np.float64) for i in range(2)]
    _, want = formulas(p, ids, labels, 2, True, masks)
    for k in alone:
        assert np.array_equal(alone[k], beside[k]), k
        assert np.linalg.norm(alone[k].ravel() - want[k].ravel()) <= 1e-4 * np.linalg.norm(want[k]), k
    ctx.close()
