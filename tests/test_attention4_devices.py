"""tr_gpu_open_device's answers for devices that are not there (as a process without GPUs sees them all)."""
import os
import subprocess
import sys


def test_devices_that_are_not_there():
    code = """
import ctypes as C
from trochilus_b200 import moe
L, err = moe.lib(), C.create_string_buffer(256)
for d in (0, 1, -1, 64, 2 ** 31 - 1):
    assert not L.tr_gpu_open_device(d, err, 256) and b"device %d is none of the 0" % d in err.value
try:
    moe.GpuAttn4(1, 1, 1, 1, 64, 64, device=3)
except RuntimeError as e:
    assert "device 3" in str(e)
else:
    raise AssertionError
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120, cwd=root, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
