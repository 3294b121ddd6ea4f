"""The scratch that group norm asks for, against what its launchers are about to write, over many problems.

The launchers compare the two before they launch anything and answer "invalid argument" where the scratch is too small. The
sweep runs in a process that sees no GPU, where a launch that may go ahead ends with another error instead; the addresses it
passes are never read."""
import os
import subprocess
import sys

import pytest

SWEEP = r"""
import ctypes, random, sys
from flagdnn_b200 import _native as nat

lib = nat.load()
rng = random.Random(int(sys.argv[1]))
SIZE = {nat.F16: 2, nat.BF16: 2, nat.F32: 4}


def refused(shape, groups, dtype, backward, shift, wide=0):
    n, c, h, w = shape
    d = nat.NormDesc()
    d.dtype = d.param_dtype = dtype
    d.n, d.c, d.h, d.w, d.groups, d.eps = n, c, h, w, groups, 1e-5
    pitch = c + wide
    for field in (d.x_strides, d.y_strides, d.dy_strides, d.dx_strides):
        field[:] = [h * w * pitch, 1, w * pitch, pitch]
    size = ctypes.c_int64()
    nat.check(lib.fdnn_group_norm_workspace_bytes(ctypes.byref(d), backward, ctypes.byref(size)))
    at = 1 << 20
    x, y, ws = at + shift * SIZE[dtype], at, at if size.value else None
    if backward:
        status = lib.fdnn_group_norm_bwd(ctypes.byref(d), x, x, at, at, at, at, y, at, at, ws, size.value, None)
    else:
        status = lib.fdnn_group_norm_fwd(ctypes.byref(d), x, at, at, y, None, None, ws, size.value, None)
    text = lib.fdnn_last_error().decode()
    assert status != nat.FDNN_OK, "a launch went ahead: this process was to have no GPU"
    return "invalid argument" in text or status == nat.FDNN_WORKSPACE_TOO_SMALL


def log(low, high):
    return int(low * (high / low) ** rng.random() + 0.5)


bad, count = [], 0
for _ in range(int(sys.argv[2])):
    per = rng.choice([1, 1, 1, 2, 3, log(1, 64), log(1, 2048)])
    groups = log(1, 64)
    if rng.random() < 0.2:
        h = w = 1
    else:
        h, w = log(1, 300), log(1, 300)
    case = ((log(1, 64), per * groups, h, w), groups, rng.choice([nat.F16, nat.BF16, nat.F32]), rng.random() < 0.5, rng.choice([0, 0, 1, 2, 4]),
            rng.choice([0, 0, 0, 1, 2, 8]))
    count += 1
    if refused(*case):
        bad.append(case)
print(count, len(bad), bad[:5])
sys.exit(1 if bad else 0)
"""


@pytest.mark.parametrize("seed", [0, 1])
def test_the_scratch_is_what_the_launchers_need(native_lib, seed):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=root)
    done = subprocess.run([sys.executable, "-c", SWEEP, str(seed), "40000"], env=env, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout + done.stderr
