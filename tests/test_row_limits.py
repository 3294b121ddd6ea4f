"""Row counts near the end of 32 bits: the kernels step past them in 32 bits, so the library takes rather fewer.

The calls are made in a process that sees no GPU; their addresses are never read."""
import os
import subprocess
import sys

CALLS = r"""
import ctypes
from flagdnn_b200 import _native as nat

lib = nat.load()
size = ctypes.c_int64()


def norm(n, h=1):
    d = nat.NormDesc()
    d.dtype = d.param_dtype = nat.BF16
    d.n, d.c, d.h, d.w, d.groups, d.eps = n, 3, h, h, 3, 1e-5
    for field in (d.x_strides, d.y_strides, d.dy_strides, d.dx_strides):
        field[:] = [3 * h * h, 1, 3 * h, 3]
    return d


def scan(n):
    d = nat.ScanDesc()
    d.dtype, d.n, d.l, d.c, d.s, d.groups = nat.BF16, n, 1, 1, 1, 1
    return d


for n in (0x7fffffff, 0x7fffffff - 1024):
    for h in (1, 2):
        for backward in (0, 1):
            assert lib.fdnn_group_norm_workspace_bytes(ctypes.byref(norm(n, h)), backward, ctypes.byref(size)) == nat.FDNN_NOT_SUPPORTED
        assert lib.fdnn_group_norm_fwd(ctypes.byref(norm(n, h)), 16, None, None, 16, None, None, 16, 1 << 60, None) == nat.FDNN_NOT_SUPPORTED
        assert lib.fdnn_group_norm_bwd(ctypes.byref(norm(n, h)), 16, 16, 16, 16, None, None, 16, None, None, 16, 1 << 60, None) == nat.FDNN_NOT_SUPPORTED
    assert lib.fdnn_selective_scan_step(ctypes.byref(scan(n)), *[16] * 5, None, None, None, 16, n, None, 16, None) == nat.FDNN_NOT_SUPPORTED
for backward in (0, 1):
    assert lib.fdnn_group_norm_workspace_bytes(ctypes.byref(norm(0x7fffffff - 65536)), backward, ctypes.byref(size)) == nat.FDNN_OK
"""


def test_rows_that_32_bits_do_not_count(native_lib):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", CALLS], env=dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=root), capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
