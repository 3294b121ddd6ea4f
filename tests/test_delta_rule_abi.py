"""The C ABI and the host functions of the gated delta rule and of mm_bias_act, as far as they go without a GPU."""
import ctypes

import pytest
import torch

import flagdnn_b200 as fd
from flagdnn_b200 import _native as nat
from oracle import delta_oracle as do


def _rule(**kw):
    d = nat.DeltaRuleDesc()
    d.dtype = d.gate_dtype = nat.BF16
    d.n, d.l, d.key_heads, d.heads, d.dk, d.dv, d.scale = 2, 100, 2, 4, 64, 64, 0.125
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _mm(**kw):
    d = nat.MmDesc()
    d.dtype, d.m, d.n, d.k = nat.BF16, 4, 64, 64
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_structures_are_the_headers(native_lib):
    assert ctypes.sizeof(nat.DeltaRuleDesc) == 12 * 4 + (4 * 4 + 2 * 3) * 8
    assert ctypes.sizeof(nat.MmDesc) == 6 * 4 + 8 * 8


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nat.F64), nat.FDNN_NOT_SUPPORTED), (dict(gate_dtype=nat.F16), nat.FDNN_NOT_SUPPORTED), (dict(n=-1), nat.FDNN_BAD_PARAM),
    (dict(l=-1), nat.FDNN_BAD_PARAM), (dict(heads=-1), nat.FDNN_BAD_PARAM), (dict(heads=3), nat.FDNN_BAD_PARAM), (dict(key_heads=0), nat.FDNN_BAD_PARAM),
    (dict(dk=0), nat.FDNN_NOT_SUPPORTED), (dict(dk=257), nat.FDNN_NOT_SUPPORTED), (dict(dv=0), nat.FDNN_NOT_SUPPORTED), (dict(dv=1025), nat.FDNN_NOT_SUPPORTED),
    (dict(heads=65536, key_heads=65536), nat.FDNN_NOT_SUPPORTED), (dict(n=0x7fffffff), nat.FDNN_NOT_SUPPORTED), (dict(l=0x7fffffff), nat.FDNN_NOT_SUPPORTED)])
def test_bad_rule_descriptors(native_lib, change, status):
    d, nbytes = _rule(**change), ctypes.c_int64()
    assert native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)) == status
    assert native_lib.fdnn_gated_delta_rule_fwd(ctypes.byref(d), *[16] * 5, None, None, None, None, 16, None, 16, 1 << 40, None) == status
    assert native_lib.fdnn_gated_delta_rule_step(ctypes.byref(d), *[16] * 5, None, None, 16, 2, None, 16, None) == status
    assert native_lib.fdnn_last_error()


def test_missing_rule_tensors_and_workspaces(native_lib):
    d, nbytes = _rule(), ctypes.c_int64()
    fwd, step = native_lib.fdnn_gated_delta_rule_fwd, native_lib.fdnn_gated_delta_rule_step
    assert fwd(None, *[16] * 5, None, None, None, None, 16, None, 16, 1 << 40, None) == nat.FDNN_BAD_PARAM
    for missing in range(5):
        given = [16] * 5
        given[missing] = None
        assert fwd(ctypes.byref(d), *given, None, None, None, None, 16, None, 16, 1 << 40, None) == nat.FDNN_BAD_PARAM
        assert step(ctypes.byref(d), *given, None, None, 16, 2, None, 16, None) == nat.FDNN_BAD_PARAM
    assert step(ctypes.byref(d), *[16] * 5, None, None, 16, 1, None, 16, None) == nat.FDNN_BAD_PARAM      # two rows, one state
    assert step(ctypes.byref(d), *[16] * 5, None, None, None, 2, None, 16, None) == nat.FDNN_BAD_PARAM
    nat.check(native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
    assert nbytes.value > 0
    assert fwd(ctypes.byref(d), *[16] * 5, None, None, None, None, 16, None, None, 0, None) == nat.FDNN_WORKSPACE_TOO_SMALL
    assert fwd(ctypes.byref(d), *[16] * 5, None, None, None, None, 16, None, 16, nbytes.value - 1, None) == nat.FDNN_WORKSPACE_TOO_SMALL
    assert fwd(ctypes.byref(d), *[16] * 5, None, None, None, None, 16, None, 8, nbytes.value, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), None) == nat.FDNN_BAD_PARAM
    for nothing in (_rule(n=0), _rule(heads=0)):
        assert fwd(ctypes.byref(nothing), *[None] * 11, None, 0, None) == nat.FDNN_OK
        nat.check(native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(nothing), ctypes.byref(nbytes)))
        assert nbytes.value == 0


def test_the_workspace_grows_with_the_chunks(native_lib):
    def size(**kw):
        d, nbytes = _rule(**kw), ctypes.c_int64()
        nat.check(native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
        return nbytes.value

    one = size(l=64)
    assert size(l=128) == 2 * one and size(l=10) == 0 and size(l=64, dk=129) == 0
    assert size(l=128 * 64, n=2000) == 1000 * 128 * one                 # rows enough for all SMs: whole
    assert size(l=128 * 64) > 128 * one                                  # few rows in segments, whose ends and starts are kept
    assert size(n=1 << 14, l=1 << 20) == one // 2 * (1 << 28)            # counted in 64 bits


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nat.F64), nat.FDNN_NOT_SUPPORTED), (dict(m=-1), nat.FDNN_BAD_PARAM), (dict(n=-1), nat.FDNN_BAD_PARAM), (dict(k=-1), nat.FDNN_BAD_PARAM),
    (dict(activation=nat.ACT_SILU), nat.FDNN_BAD_PARAM), (dict(activation=-1), nat.FDNN_BAD_PARAM), (dict(m=(1 << 22) + 1), nat.FDNN_NOT_SUPPORTED),
    (dict(n=0x7fffffff), nat.FDNN_NOT_SUPPORTED), (dict(k=0x7fffffff), nat.FDNN_NOT_SUPPORTED)])
def test_bad_product_descriptors(native_lib, change, status):
    d, yes = _mm(**change), ctypes.c_int32()
    assert native_lib.fdnn_mm_rows_preferred(ctypes.byref(d), ctypes.byref(yes)) == status
    assert native_lib.fdnn_mm_rows_fwd(ctypes.byref(d), 16, 16, None, None, 16, None) == status


def test_missing_product_tensors(native_lib):
    d = _mm()
    for given in ((None, 16, 16), (16, None, 16), (16, 16, None)):
        assert native_lib.fdnn_mm_rows_fwd(ctypes.byref(d), given[0], given[1], None, None, given[2], None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_mm_rows_fwd(None, 16, 16, None, None, 16, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_mm_rows_preferred(ctypes.byref(d), None) == nat.FDNN_BAD_PARAM
    for nothing in (_mm(m=0), _mm(n=0)):
        assert native_lib.fdnn_mm_rows_fwd(ctypes.byref(nothing), None, None, None, None, None, None) == nat.FDNN_OK


def test_which_products_are_of_few_rows(native_lib):
    def preferred(**kw):
        d, yes = _mm(**kw), ctypes.c_int32()
        nat.check(native_lib.fdnn_mm_rows_preferred(ctypes.byref(d), ctypes.byref(yes)))
        return bool(yes.value)

    assert preferred(m=1, n=8192, k=64) and preferred(m=16, n=8192, k=64) and preferred(m=500, n=8192, k=7)
    assert preferred(m=64, n=2048, k=4096) and not preferred(m=65, n=2048, k=4096) and preferred(m=256, n=512, k=8192)
    assert not preferred(m=64, n=4096, k=2048) and not preferred(m=48, n=1024, k=1024)
    assert preferred(m=1024, n=16, k=8192) and not preferred(m=1025, n=16, k=8192) and not preferred(m=513, n=16, k=2048)
    assert preferred(m=5000, n=8192, k=64, dtype=nat.F32)      # whose sums a convolution keeps in one accumulator


def test_cpu_tensors_are_refused():
    q, v, gate, state = torch.randn(2, 5, 1, 8), torch.randn(2, 5, 2, 8), torch.randn(2, 5, 2), torch.zeros(2, 2, 8, 8)
    for call in (lambda: fd.gated_delta_rule(q, q, v, gate, gate), lambda: fd.gated_delta_rule_step(q[:, 0], q[:, 0], v[:, 0], gate[:, 0], gate[:, 0], state),
                 lambda: fd.mm_bias_act(q[0, :, 0], torch.randn(8, 3))):
        with pytest.raises(NotImplementedError, match="requires CUDA input"):
            call()


def test_the_oracle_agrees_with_the_chunks_formulas():
    """Two ways to the same numbers: token by token, and a chunk solved at once."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    length, dk, dv = 12, 6, 5
    q, k, v, before = r(1, length, 1, dk), r(1, length, 1, dk) * 0.4, r(1, length, 1, dv), r(1, 1, dv, dk)
    decay, beta = -torch.rand(1, length, 1, generator=g, dtype=torch.float64), torch.rand(1, length, 1, generator=g, dtype=torch.float64)
    want = do.gated_delta_rule(q, k, v, decay, beta, scale=1.0, initial_state=before)
    k, q, v, s, total, b = k[0, :, 0], q[0, :, 0], v[0, :, 0], before[0, 0], decay[0, :, 0].cumsum(0), beta[0, :, 0]
    between = torch.exp(total[:, None] - total)
    a = torch.tril(b[:, None] * between * (k @ k.T), -1)
    u = torch.linalg.solve(torch.eye(length, dtype=torch.float64) + a, b[:, None] * (v - total.exp()[:, None] * (k @ s.T)))
    y = total.exp()[:, None] * (q @ s.T) + torch.tril(between * (q @ k.T)) @ u
    end = total[-1].exp() * s + (between[-1][:, None] * u).T @ k
    torch.testing.assert_close(y, want.y[0, :, 0], rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(end, want.state[0, 0], rtol=1e-10, atol=1e-12)
    assert (want.y.abs() <= want.y_size + 1e-12).all() and (want.state.abs() <= want.state_size + 1e-12).all()


def test_the_oracle_reads_its_options():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 7, h, 4, generator=g, dtype=torch.float64) for h in (1, 1, 3))
    raw_delta, raw_beta = torch.randn(2, 7, 3, generator=g, dtype=torch.float64), torch.randn(2, 7, 3, generator=g, dtype=torch.float64)
    A, bias = -torch.rand(3, generator=g, dtype=torch.float64), torch.randn(3, generator=g, dtype=torch.float64)
    normed = [t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k)]
    ready = do.gated_delta_rule(*(t.repeat_interleave(3, 2) for t in normed), v, A * torch.nn.functional.softplus(raw_delta + bias, threshold=1000),
                                torch.sigmoid(raw_beta), lengths=[7, 4])
    raw = do.gated_delta_rule(q, k, v, raw_delta, raw_beta, A, bias, True, True, True, lengths=[7, 4])
    torch.testing.assert_close(raw.y, ready.y, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(raw.state, ready.state, rtol=1e-12, atol=1e-12)
    assert not raw.y[1, 4:].any()
