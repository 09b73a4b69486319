"""The first call of a process may be one that is captured: the status block is made while a capture is under way."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
import torch
import cfk_b200 as cfk
lib = cfk.load()
which, mode = sys.argv[1:]
q, s = torch.ones(4, 64, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda")
w = torch.full((64, 64), 2, dtype=torch.int8, device="cuda")
x, v = torch.ones(128, 64, dtype=torch.float16, device="cuda"), torch.ones(128, 64, dtype=torch.float16, device="cuda")
y, z = torch.zeros(4, 64, device="cuda"), torch.zeros(128, 128, dtype=torch.float16, device="cuda")
stream = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream, capture_error_mode=mode):
    if which == "gemm_i8":
        lib.gemm_i8(q, w, y, m=4, n=64, k=64, out_dtype=cfk.FP32, a_scale=s, b_scale=s, stream=stream.cuda_stream)
    else:
        lib.gemm(x, v, z, dtype=cfk.FP16, m=128, n=128, k=64, stream=stream.cuda_stream)
for _ in range(2):
    y.zero_(), z.zero_()
    graph.replay()
    lib.check_device()
    got = y if which == "gemm_i8" else z
    assert bool((got == (128.0 if which == "gemm_i8" else 64.0)).all()), got
assert lib.selftest_wait_gives_up(20) == 0          # the block works: a wait that gives up is reported, and the next replay runs
assert lib.device_status() == (6, 901)
graph.replay()
lib.check_device()
print("captured")
"""


@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
@pytest.mark.parametrize("which", ["gemm_i8", "gemm"])
def test_the_first_call_may_be_captured(cuda, which, mode):
    import cfk_b200
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(cfk_b200.__file__))))
    r = subprocess.run([sys.executable, "-c", PROGRAM, which, mode], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
