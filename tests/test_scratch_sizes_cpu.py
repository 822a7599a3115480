"""lh_scratch_bytes answers for any sizes: it is asked before a call checks its own."""

import subprocess
import sys

import pytest

from linghe_b200 import _lib

KINDS = ["rmsnorm_bwd", "batch_silu_bwd", "smooth_quant", "smooth_quant_bwd", "row_id_map", "rmsnorm_pair_bwd", "rmsnorm_gemm", "none of them"]


@pytest.mark.parametrize("kind", KINDS)
def test_any_sizes(kind):
    """In a process of its own, which an integer division by zero would end."""
    code = f"""
import ctypes
size = ctypes.CDLL({_lib.LIB_PATH!r}).lh_scratch_bytes
size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_char_p, ctypes.c_int64, ctypes.c_int64]
for rows in (-1, 0, 1, 4, 1 << 20, (1 << 31) - 1):
    for cols in (-128, -1, 0, 1, 8, 15, 16, 31, 100, 128, 200, 4096, 5120, 8192, 8320, 1 << 20):
        v = size({kind!r}.encode(), rows, cols)
        if {kind!r} == "rmsnorm_pair_bwd":
            assert (v > 0) == (rows > 0 and cols in (128, 4096, 5120, 8192)), (rows, cols, v)
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), (r.returncode, r.stderr[-500:])
