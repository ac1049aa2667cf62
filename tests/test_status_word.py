"""The witness calls' status word: made without allocating or waiting, on every device that grape_init takes.  On a runtime that
only keeps count (tests/native/fake_hip.cpp, linked in front of HIP's), and under a capture on the GPU."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
NATIVE = os.path.join(HERE, "native")
PKG = os.path.join(os.path.dirname(HERE), "grape_amd")


def test_init_and_witness_calls_on_any_device_without_memory(tmp_path):
    fake, exe = str(tmp_path / "libfake_hip.so"), str(tmp_path / "status_word")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", fake, os.path.join(NATIVE, "fake_hip.cpp")])
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", exe, os.path.join(NATIVE, "status_word.cpp"),
                           "-Wl,--no-as-needed", "-Wl,--export-dynamic", "-L" + str(tmp_path), "-lfake_hip", "-L" + PKG, "-lgrape_hip", "-Wl,-rpath," + str(tmp_path), "-Wl,-rpath," + PKG])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


INIT_CAPTURED = """
import numpy as np, torch
from grape_amd import ops
from oracle import witness_oracle as wo
rng = np.random.default_rng(1)
x, w = rng.integers(-1000, 1000, (1, 100)).astype(np.int32), rng.integers(0, 256, (40, 50)).astype(np.uint8)
scales = rng.integers(-400, 400, (40, 4)).astype(np.int32)
dx, dw, ds = (torch.from_numpy(a).cuda() for a in (x, w, scales))
q, r = torch.zeros((1, 40), dtype=torch.int32, device="cuda"), torch.zeros((1, 40), dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                                    # in global mode, on a stream of its own
    ops.wit_matvec_q4(dx, dw, ds, 32, q=q, r=r)                  # calls grape_init
want = wo.matvec_q4(x, w, scales, 32, None)
for _ in range(3):
    q.fill_(-1), r.fill_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(q.cpu().numpy(), want[0]) and np.array_equal(r.cpu().numpy(), want[1])
    assert ops.wit_status() == 0
ops.wit_matvec_q4(dx, dw, ds * 1000000, 32, scale=1)
assert ops.wit_status() == 1 and ops.wit_status() == 0
print("captured")
"""


@pytest.mark.gpu
def test_grape_init_while_a_stream_is_captured():
    res = subprocess.run([sys.executable, "-c", INIT_CAPTURED], cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and "captured" in res.stdout, res.stdout + res.stderr
