"""Which of up to 16 rows go to the kernel of few rows, by the figures at fdnn_mm_rows_preferred's rule (no GPU needed: 148 SMs)."""
import ctypes

import pytest

from flagdnn_b200 import _native as nat


@pytest.mark.parametrize("m,k,n,act,few", [
    (8, 4096, 8192, nat.ACT_NONE, True), (15, 4096, 8192, nat.ACT_NONE, True), (16, 4096, 4096, nat.ACT_NONE, True), (16, 4096, 6144, nat.ACT_NONE, True),
    (16, 4096, 8192, nat.ACT_NONE, False), (16, 4096, 8192, nat.ACT_RELU, False), (16, 4096, 8192, nat.ACT_GELU, True),
    (16, 4096, 8192, nat.ACT_GELU_TANH, True), (16, 4096, 12288, nat.ACT_NONE, True), (16, 8192, 8192, nat.ACT_NONE, False),
    (16, 2048, 8192, nat.ACT_NONE, True), (4, 512, 24576, nat.ACT_NONE, True), (8, 512, 24576, nat.ACT_NONE, False),
    (16, 4096, 8188, nat.ACT_NONE, True), (8, 512, 24577, nat.ACT_NONE, True), (16, 256, 18944, nat.ACT_GELU, True), (16, 256, 18952, nat.ACT_GELU, False), (8, 1024, 24576, nat.ACT_NONE, True)])
def test_up_to_sixteen_rows(native_lib, m, k, n, act, few):
    def preferred(dtype=nat.BF16, a=(k, 1), b=(n, 1)):
        d, yes = nat.MmDesc(), ctypes.c_int32()
        d.dtype, d.m, d.n, d.k, d.activation = dtype, m, n, k, act
        d.a_strides[:], d.b_strides[:] = a, b
        nat.check(native_lib.fdnn_mm_rows_preferred(ctypes.byref(d), ctypes.byref(yes)))
        return bool(yes.value)

    assert preferred() == preferred(nat.F16) == preferred(b=(1, k)) == preferred(a=(k + 64, 1)) == few
    # what the convolution would lay out anew, and fp32
    assert preferred(a=(1, m)) and preferred(a=(k + 1, 1)) and preferred(b=(n + 4, 1)) and preferred(b=(1, k + 1)) and preferred(nat.F32)
