"""How long a context lives: until it is destroyed and its last tensor is freed, in either
order.  Python's collector takes a Device and its QTensors that share a cycle in any order,
and a tensor's release must not read a context that is gone.

The library itself runs here without a GPU, in a process of its own where the HIP calls it
makes are tests/lifetime/host_hip.cpp (two devices of host memory) and freed host memory is
overwritten (MALLOC_PERTURB_), so that a read of a freed context gives no device's number."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

PRELUDE = """
import ctypes, gc, sys
gc.disable()
hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from mold_amd import Device, GgmlDType, QTensor, _lib

class Stream:
    cuda_stream = 0

class Blocks:
    def __init__(self, n):
        self.host = (ctypes.c_float * n)(*range(n))
    def data_ptr(self): return ctypes.addressof(self.host)
    def numel(self): return len(self.host)
    def element_size(self): return 4

def tensor(dev, n=64):
    return QTensor.from_device_blocks(dev, GgmlDType.F32, (1, n), Blocks(n), Stream())

def done():
    gc.collect()
    assert (hip.host_hip_bad_devices(), hip.host_hip_bad_frees(), hip.host_hip_live()) == (0, 0, 0), (
        hip.host_hip_bad_devices(), hip.host_hip_bad_frees(), hip.host_hip_live())
    print("ok")
"""


@pytest.fixture(scope="module")
def host_hip(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("host_hip") / "libhost_hip.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "lifetime", "host_hip.cpp"), "-o", out], check=True)
    return out


def _run(host_hip, code):
    r = subprocess.run([sys.executable, "-c", PRELUDE + code, host_hip], cwd=ROOT, capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, MALLOC_PERTURB_="165"))
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("ordinal", [0, 1])
def test_tensor_outlives_the_context(host_hip, ordinal):
    """mq_ctx_destroy before the last mq_qtensor_free, and after it."""
    _run(host_hip, f"""
dev = Device({ordinal})
a, b = tensor(dev), tensor(dev)
a.free()
dev.close()
b.free()
dev = Device({ordinal})
a = tensor(dev)
a.free()
dev.close()
done()
""")


def test_collected_together(host_hip):
    """A cycle that holds a Device and its tensors, as an exception's frame does."""
    _run(host_hip, """
for first in (True, False):
    class Holder:
        pass
    h = Holder()
    h.me = h
    h.dev = Device(1)
    h.tensors = [tensor(h.dev) for _ in range(3)]
    if first:
        h.dev.back = h
    else:
        for t in h.tensors:
            t.back = h
    del h, Holder
    t = None
    gc.collect()
done()
""")


def test_arena_outlives_the_context(host_hip):
    """Tensors in an arena beside one that no longer fits it."""
    _run(host_hip, """
dev = Device(1)
dev.reserve_arena(2048)
ts = [tensor(dev, n) for n in (64, 256, 4096)]
dev.close()
assert hip.host_hip_live() == 2
while ts:
    ts.pop(0).free()
done()
""")
