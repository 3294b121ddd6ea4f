"""The C ABI and the host functions of group norm and the state space operators, as far as they go without a GPU."""
import ctypes

import pytest
import torch

import flagdnn_b200 as fd
from flagdnn_b200 import _native as nat
from oracle import sequence_oracle as so


def _norm(**kw):
    d = nat.NormDesc()
    d.dtype = d.param_dtype = nat.BF16
    d.n, d.c, d.h, d.w, d.groups, d.eps = 2, 64, 8, 8, 8, 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _conv(**kw):
    d = nat.CausalConvDesc()
    d.dtype, d.n, d.l, d.c, d.width = nat.BF16, 2, 5, 64, 4
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _scan(**kw):
    d = nat.ScanDesc()
    d.dtype, d.n, d.l, d.c, d.s, d.groups = nat.BF16, 2, 5, 64, 16, 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_structures_are_the_headers(native_lib):
    assert ctypes.sizeof(nat.NormDesc) == 10 * 4 + 16 * 8
    assert ctypes.sizeof(nat.CausalConvDesc) == 6 * 4 + 6 * 8
    assert ctypes.sizeof(nat.ScanDesc) == 8 * 4 + (4 * 3 + 2 * 4) * 8


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nat.F64), nat.FDNN_NOT_SUPPORTED), (dict(dtype=9), nat.FDNN_NOT_SUPPORTED), (dict(param_dtype=nat.F16), nat.FDNN_NOT_SUPPORTED),
    (dict(groups=0), nat.FDNN_BAD_PARAM), (dict(groups=7), nat.FDNN_BAD_PARAM), (dict(c=0), nat.FDNN_BAD_PARAM), (dict(n=-1), nat.FDNN_BAD_PARAM),
    (dict(activation=5), nat.FDNN_BAD_PARAM), (dict(activation=-1), nat.FDNN_BAD_PARAM), (dict(eps=-1.0), nat.FDNN_BAD_PARAM),
    (dict(eps=float("nan")), nat.FDNN_BAD_PARAM)])
def test_bad_norm_descriptors(native_lib, change, status):
    nbytes = ctypes.c_int64()
    d = _norm(**change)
    assert native_lib.fdnn_group_norm_workspace_bytes(ctypes.byref(d), 0, ctypes.byref(nbytes)) == status
    assert native_lib.fdnn_group_norm_fwd(ctypes.byref(d), 16, 16, 16, 16, None, None, 16, 1 << 40, None) == status
    assert native_lib.fdnn_group_norm_bwd(ctypes.byref(d), 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 1 << 40, None) == status
    assert native_lib.fdnn_last_error()


def test_missing_norm_tensors_and_workspaces(native_lib):
    d, nbytes = _norm(), ctypes.c_int64()
    fwd, bwd = native_lib.fdnn_group_norm_fwd, native_lib.fdnn_group_norm_bwd
    assert fwd(None, 16, None, None, 16, None, None, None, 0, None) == nat.FDNN_BAD_PARAM
    assert fwd(ctypes.byref(d), None, None, None, 16, None, None, None, 0, None) == nat.FDNN_BAD_PARAM
    assert fwd(ctypes.byref(d), 16, None, None, 16, 16, None, None, 0, None) == nat.FDNN_BAD_PARAM     # mean without rstd
    assert bwd(ctypes.byref(d), 16, 16, None, 16, None, None, 16, None, None, None, 0, None) == nat.FDNN_BAD_PARAM
    nat.check(native_lib.fdnn_group_norm_workspace_bytes(ctypes.byref(d), 1, ctypes.byref(nbytes)))
    assert nbytes.value > 0
    assert bwd(ctypes.byref(d), 16, 16, 16, 16, None, None, 16, None, None, None, 0, None) == nat.FDNN_WORKSPACE_TOO_SMALL
    assert bwd(ctypes.byref(d), 16, 16, 16, 16, None, None, 16, None, None, 8, nbytes.value, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_group_norm_workspace_bytes(ctypes.byref(d), 1, None) == nat.FDNN_BAD_PARAM
    nothing = _norm(n=0)
    assert fwd(ctypes.byref(nothing), None, None, None, None, None, None, None, 0, None) == nat.FDNN_OK


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nat.F64), nat.FDNN_NOT_SUPPORTED), (dict(width=0), nat.FDNN_NOT_SUPPORTED), (dict(width=9), nat.FDNN_NOT_SUPPORTED),
    (dict(l=-1), nat.FDNN_BAD_PARAM), (dict(activation=7), nat.FDNN_BAD_PARAM)])
def test_bad_convolution_descriptors(native_lib, change, status):
    d = _conv(**change)
    assert native_lib.fdnn_causal_conv1d_fwd(ctypes.byref(d), 16, 16, None, None, None, 16, None, None) == status
    d.l = 1 if d.l > 0 else d.l
    assert native_lib.fdnn_causal_conv1d_step(ctypes.byref(d), 16, 16, None, 16, 2, None, 16, None) == status


def test_missing_convolution_tensors(native_lib):
    d = _conv()
    assert native_lib.fdnn_causal_conv1d_fwd(ctypes.byref(d), None, 16, None, None, None, 16, None, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_causal_conv1d_fwd(ctypes.byref(d), 16, None, None, None, None, 16, None, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_causal_conv1d_step(ctypes.byref(d), 16, 16, None, 16, 1, None, 16, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_causal_conv1d_step(ctypes.byref(d), 16, 16, None, None, 2, None, 16, None) == nat.FDNN_BAD_PARAM


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nat.F64), nat.FDNN_NOT_SUPPORTED), (dict(s=0), nat.FDNN_NOT_SUPPORTED), (dict(s=257), nat.FDNN_NOT_SUPPORTED),
    (dict(groups=3), nat.FDNN_BAD_PARAM), (dict(groups=0), nat.FDNN_BAD_PARAM), (dict(c=-1), nat.FDNN_BAD_PARAM)])
def test_bad_scan_descriptors(native_lib, change, status):
    d, nbytes = _scan(**change), ctypes.c_int64()
    assert native_lib.fdnn_selective_scan_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)) == status
    assert native_lib.fdnn_selective_scan_fwd(ctypes.byref(d), *[16] * 5, None, None, None, None, None, 16, None, 16, 1 << 40, None) == status
    assert native_lib.fdnn_selective_scan_step(ctypes.byref(d), *[16] * 5, None, None, None, 16, 2, None, 16, None) == status


def test_missing_scan_tensors(native_lib):
    d = _scan()
    for missing in range(5):
        given = [16] * 5
        given[missing] = None
        assert native_lib.fdnn_selective_scan_fwd(ctypes.byref(d), *given, None, None, None, None, None, 16, None, 16, 1 << 40, None) == nat.FDNN_BAD_PARAM
        assert native_lib.fdnn_selective_scan_step(ctypes.byref(d), *given, None, None, None, 16, 2, None, 16, None) == nat.FDNN_BAD_PARAM
    assert native_lib.fdnn_selective_scan_step(ctypes.byref(d), *[16] * 5, None, None, None, 16, 1, None, 16, None) == nat.FDNN_BAD_PARAM


def test_cpu_tensors_are_refused():
    x, w = torch.randn(2, 5, 8), torch.randn(8, 4)
    a, bc = -torch.rand(8, 4), torch.randn(2, 5, 4)
    for call in (lambda: fd.group_norm(x.transpose(1, 2), 4), lambda: fd.causal_conv1d(x, w), lambda: fd.selective_scan(x, x, a, bc, bc),
                 lambda: fd.causal_conv1d_step(x[:, 0], torch.zeros(2, 3, 8), w),
                 lambda: fd.selective_scan_step(x[:, 0], x[:, 0], a, bc[:, 0], bc[:, 0], torch.zeros(2, 8, 4))):
        with pytest.raises(NotImplementedError, match="requires CUDA input"):
            call()


def test_group_norm_is_captured():
    x, w = fd.TensorSpec("x", (2, 8, 4, 4), torch.float32), fd.TensorSpec("w", (8,), torch.float32)

    @fd.graph
    def block(x, w):
        return fd.group_norm(x, 4, weight=w, activation="silu")

    compiled = fd.compile(block, inputs=[x, w], options={"cache": None})
    node, = compiled.graph.nodes
    assert node.op_type == "group_norm" and node.attrs["operands"] == ("weight",) and node.attrs["activation"] == "silu"

    def stats(x, w):
        return fd.group_norm(x, 4, return_stats=True)

    def uneven(x, w):
        return fd.group_norm(x, 3)

    with pytest.raises(NotImplementedError, match="values only"):
        fd.compile(stats, inputs=[x, w], options={"cache": None})
    with pytest.raises(RuntimeError, match="divisible"):
        fd.compile(uneven, inputs=[x, w], options={"cache": None})


def test_the_oracle_agrees_with_torch():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 12, 5, generator=g, dtype=torch.float64, requires_grad=True)
    w, b = (torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    dy = torch.randn(3, 12, 5, generator=g, dtype=torch.float64)
    for act, fn in (("none", lambda v: v), ("relu", torch.relu), ("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu),
                    ("gelu_tanh", lambda v: torch.nn.functional.gelu(v, approximate="tanh"))):
        y = fn(torch.nn.functional.group_norm(x, 4, w, b))
        torch.testing.assert_close(so.group_norm(x, 4, w, b, act=act)[0], y.detach(), rtol=1e-12, atol=1e-12)
        for got, want in zip(so.group_norm_grad(dy, x, 4, w, b, act=act), torch.autograd.grad(y, (x, w, b), dy)):
            torch.testing.assert_close(got, want, rtol=1e-10, atol=1e-10)
    seq, f = torch.randn(2, 9, 6, generator=g, dtype=torch.float64), torch.randn(6, 3, generator=g, dtype=torch.float64)
    y = torch.nn.functional.conv1d(torch.nn.functional.pad(seq.transpose(1, 2), (2, 0)), f[:, None], groups=6).transpose(1, 2)
    torch.testing.assert_close(so.causal_conv1d(seq, f)[0], y, rtol=1e-12, atol=1e-12)
