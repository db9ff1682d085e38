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
