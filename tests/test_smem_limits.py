"""A kernel's limit of dynamic shared memory is one number for the whole process: it may not depend on a call."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "musapy_b200", "csrc")


def test_shared_memory_limits_are_constants():
    """Every limit that is set is a constant by its name (kName or NAME), not a call's size: two host threads that set
    their own sizes in turn would have each other's launches refused."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        for m in re.finditer(r"cudaFuncAttributeMaxDynamicSharedMemorySize,\s*([^)]*)\)", text):
            found += 1
            assert re.fullmatch(r"k[A-Z]\w*|[A-Z][A-Z0-9_]*", m.group(1).strip()), f"{name}: limit {m.group(1)!r}"
    assert found >= 3


# Eight threads, each the first to call with its length of rows and so its need of shared memory.
THREADS = r'''
import ctypes
import sys
import threading

import torch

from musapy_b200._lib import LIB, last_error

vp, i64, f64, sz, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t, ctypes.c_int
LIB.mpb_policy_loss.argtypes = [i64, i64, vp, i32, i64, vp, i32, vp, vp, vp, vp, f64, f64, f64, f64, vp, vp, vp, vp, vp, vp, sz, vp]
LIB.mpb_policy_loss.restype = i32
F32 = 10
made = []
for V in (425984, 140000, 400001, 200000, 11000, 300000, 16000, 350000):
    N = 4
    t = {"z": torch.randn(N, V, device="cuda"), "t": torch.zeros(N, dtype=torch.int64, device="cuda"),
         "f": torch.zeros(N, device="cuda"), "out": torch.zeros(64, device="cuda"), "g": torch.empty(N, V, device="cuda"),
         "s": torch.empty(64, device="cuda"), "stream": torch.cuda.Stream()}
    made.append((N, V, t))
torch.cuda.synchronize()
gate, bad = threading.Barrier(len(made)), []


def work(N, V, t):
    o = t["out"].data_ptr()
    torch.cuda.set_device(0)
    gate.wait()
    for _ in range(20):
        rc = LIB.mpb_policy_loss(N, V, t["z"].data_ptr(), F32, V, t["t"].data_ptr(), 4, t["f"].data_ptr(), t["f"].data_ptr(), None,
                                 None, 0.2, 0.2, 0.0, 1.0, o, o + 16, o + 64, o + 128, t["g"].data_ptr(), t["s"].data_ptr(), 256,
                                 t["stream"].cuda_stream)
        if rc:
            bad.append((V, rc, last_error()))


threads = [threading.Thread(target=work, args=m) for m in made]
for th in threads:
    th.start()
for th in threads:
    th.join()
torch.cuda.synchronize()
print("failed:", len(bad), bad[:3])
sys.exit(1 if bad else 0)
'''


@pytest.mark.gpu
def test_first_calls_from_several_threads(ms):
    """Each time in a new process, as the limits are set by a process's first calls."""
    for _ in range(3):
        run = subprocess.run([sys.executable, "-c", THREADS], cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, run.stdout + run.stderr[-2000:]
