"""The operators' cases as a program runs them: on inputs that are still being made, and from several threads."""
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
CASE = '{"name": "d", "op": "dropout", "count": 1 << 20, "residual": True, "p": 0.25, "train": True}'


def in_a_process(body):
    code = f"""
import threading
import torch
from neuralrs_b200 import _lib, cuda                    # (ahead of the clock)
from perf import operators
cuda.Context(0).sync()
case = {CASE}

def one(seed):
    state = operators.prepare(case, seed)
    torch.cuda._sleep(1_000_000_000)                      # (some half a second, in which the inputs are not ready)
    for name in ("x", "residual", "g"):
        state[name].neg_()
    operators.own = True
    got = operators.run(state)
    torch.cuda.synchronize()
    operators.own = False
    want = operators.run(state)
    torch.cuda.synchronize()
    for k in want:
        assert torch.equal(got[k] == 0, want[k] == 0) and float((got[k] - want[k]).abs().max()) < 1e-5, k

{body}
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=pathlib.Path(__file__).parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "Error" not in done.stderr, done.stderr[-2000:]


def test_the_first_call_waits_for_its_inputs():
    in_a_process("one(1)")


def test_a_second_thread():
    in_a_process("""
one(1)
t = threading.Thread(target=one, args=(2,))
t.start()
t.join()
one(3)
""")
