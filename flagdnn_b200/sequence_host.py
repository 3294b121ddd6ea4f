"""Host side of the state space operators: the short causal convolution and the selective scan, over prompts and for
single tokens.

Sequences are ``[N, L, C]``, tokens in order with their channels together, as ``mm`` leaves them (any strides are taken; a
slice of the columns of a wider projection needs no copy).  ``lengths`` (int32 [N]) makes a batch ragged: tokens from
``lengths[n]`` on are padding, are never read and give zeros.  States are the caller's: the convolution's is the last
``width - 1`` inputs, ``[N, width - 1, C]`` in the inputs' type, the scan's ``[N, C, S]`` float32.  The step functions update a
cache of states in place, at ``slots`` (int32 [N]; a slot outside the cache marks an idle row, whose output is zero; two rows
must not share one); it counts as written for autograd's check of saved tensors.  These are operators of the forward pass:
tensors that ask for a gradient, or carry a tangent, are refused.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _native as nat
from . import conv_host as _conv
from .norm_host import _DTYPE_IDS, activation_id, address, answered, refuse_grad, workspace

MAX_WIDTH, MAX_STATES = 8, 256


def _check_input(what: str, name: str, x: torch.Tensor, dims: int) -> None:
    if x.dim() != dims:
        raise RuntimeError(f"{what}: {name} must have {dims} dimensions, got {x.dim()}")
    if x.dtype not in _DTYPE_IDS:
        raise NotImplementedError(f"flag_dnn {what} does not support dtype={x.dtype}")
    if not x.is_cuda:
        raise NotImplementedError(f"flag_dnn {what} CUDA implementation requires CUDA input")
    if max(x.shape) > 0x7fffffff:
        raise RuntimeError(f"{what}: an extent is too large")


def _check_like(what: str, name: str, t: Optional[torch.Tensor], shape: tuple, dtype: torch.dtype, device: torch.device) -> None:
    if t is None:
        return
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise RuntimeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} must be on {device}, got {t.device}")


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


def _set(field, strides) -> None:
    for i, s in enumerate(strides):
        field[i] = s


def _check_conv(what: str, x, weight, bias):
    c = x.shape[-1]
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight[:, 0]                       # a depthwise conv1d's [C, 1, width]
    if weight.dim() != 2 or weight.shape[0] != c:
        raise RuntimeError(f"{what}: weight must have shape ({c}, width), got {tuple(weight.shape)}")
    width = weight.shape[1]
    if not 1 <= width <= MAX_WIDTH:
        raise NotImplementedError(f"flag_dnn {what} takes filters of 1 to {MAX_WIDTH} taps, got {width}")
    _check_like(what, "weight", weight, (c, width), x.dtype, x.device)
    _check_like(what, "bias", bias, (c,), x.dtype, x.device)
    return weight.contiguous(), _dense(bias), width


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
                  initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                  return_final_state: bool = False):
    """``y[n, t, c] = activation(bias[c] + sum_j weight[c, j] xs[n, t + j, c])`` where ``xs`` is ``initial_state`` (zeros if
    None) followed by ``x`` [N, L, C].  With ``return_final_state`` the result is ``(y, state after the row)``."""
    what = "causal_conv1d"
    act = activation_id(activation)
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.causal_conv1d(x, weight, bias, act, initial_state, lengths, bool(return_final_state))
        if y is not None:
            return answered(y)
    _check_input(what, "x", x, 3)
    weight, bias, width = _check_conv(what, x, weight, bias)
    n, length, c = x.shape
    _check_like(what, "initial_state", initial_state, (n, width - 1, c), x.dtype, x.device)
    _check_like(what, "lengths", lengths, (n,), torch.int32, x.device)
    refuse_grad(what, x, weight, bias, initial_state)
    initial_state, lengths = _dense(initial_state), _dense(lengths)
    y = torch.empty((n, length, c), dtype=x.dtype, device=x.device)
    final = torch.empty((n, width - 1, c), dtype=x.dtype, device=x.device) if return_final_state else None
    d = nat.CausalConvDesc()
    d.dtype, d.n, d.l, d.c, d.width, d.activation = _DTYPE_IDS[x.dtype], n, length, c, width, act
    _set(d.x_strides, x.stride())
    _set(d.y_strides, y.stride())
    with torch.cuda.device(x.device):
        nat.check(nat.load().fdnn_causal_conv1d_fwd(
            ctypes.byref(d), x.data_ptr(), weight.data_ptr(), address(bias), address(initial_state), address(lengths), y.data_ptr(),
            address(final), torch.cuda.current_stream().cuda_stream))
    return (y, final) if return_final_state else y


def _check_cache(what: str, name: str, state: torch.Tensor, tail: tuple, dtype, x: torch.Tensor, slots) -> None:
    if state.dim() != 1 + len(tail):
        raise RuntimeError(f"{what}: {name} must have {1 + len(tail)} dimensions, got {state.dim()}")
    _check_like(what, name, state, (state.shape[0], *tail), dtype, x.device)
    if not state.is_contiguous():
        raise RuntimeError(f"{what}: {name} is updated in place and must be contiguous")
    _check_like(what, "slots", slots, (x.shape[0],), torch.int32, x.device)
    if slots is None and state.shape[0] < x.shape[0]:
        raise RuntimeError(f"{what}: {state.shape[0]} states for {x.shape[0]} rows")
    if state.shape[0] > 0x7fffffff:
        raise RuntimeError(f"{what}: an extent is too large")


def causal_conv1d_step(x: torch.Tensor, conv_state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       activation: str = "none", slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``causal_conv1d`` of the next token of each row, ``x`` [N, C]; ``conv_state`` [slots, width - 1, C] is updated in place."""
    what = "causal_conv1d_step"
    act = activation_id(activation)
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.causal_conv1d_step(x, conv_state, weight, bias, act, slots)
        if y is not None:
            return answered(y)
    _check_input(what, "x", x, 2)
    weight, bias, width = _check_conv(what, x, weight, bias)
    n, c = x.shape
    _check_cache(what, "conv_state", conv_state, (width - 1, c), x.dtype, x, slots)
    refuse_grad(what, x, weight, bias, conv_state)
    slots = _dense(slots)
    y = torch.empty((n, c), dtype=x.dtype, device=x.device)
    d = nat.CausalConvDesc()
    d.dtype, d.n, d.l, d.c, d.width, d.activation = _DTYPE_IDS[x.dtype], n, 1, c, width, act
    _set(d.x_strides, (x.stride(0), 0, x.stride(1)))
    _set(d.y_strides, (c, 0, 1))
    with torch.cuda.device(x.device):
        nat.check(nat.load().fdnn_causal_conv1d_step(
            ctypes.byref(d), x.data_ptr(), weight.data_ptr(), address(bias), conv_state.data_ptr(), conv_state.shape[0],
            address(slots), y.data_ptr(), torch.cuda.current_stream().cuda_stream))
    increment_version(conv_state)
    return y


def _check_scan(what: str, u, delta, A, B, C, D, z, delta_bias):
    """The descriptor for these tensors, and them as the library takes them (B and C with their group dimension)."""
    rows, c = tuple(u.shape[:-1]), u.shape[-1]
    if A.dim() != 2 or A.shape[0] != c:
        raise RuntimeError(f"{what}: A must have shape ({c}, states), got {tuple(A.shape)}")
    s = A.shape[1]
    if not 1 <= s <= MAX_STATES:
        raise NotImplementedError(f"flag_dnn {what} takes 1 to {MAX_STATES} states a channel, got {s}")
    B = B.unsqueeze(-2) if B.dim() == u.dim() else B
    C = C.unsqueeze(-2) if C.dim() == u.dim() else C
    groups = B.shape[-2] if B.dim() == u.dim() + 1 else 0
    if groups < 1 or c % groups != 0:
        raise RuntimeError(f"{what}: B must have shape {(*rows, s)} or {(*rows, 'groups', s)} with groups dividing {c}, "
                           f"got {tuple(B.shape)}")
    for name, t, shape in (("delta", delta, u.shape), ("B", B, (*rows, groups, s)), ("C", C, (*rows, groups, s)), ("z", z, u.shape)):
        _check_like(what, name, t, shape, u.dtype, u.device)
    for name, t, shape in (("A", A, (c, s)), ("D", D, (c,)), ("delta_bias", delta_bias, (c,))):
        _check_like(what, name, t, shape, torch.float32, u.device)
    d = nat.ScanDesc()
    d.dtype, d.c, d.s, d.groups = _DTYPE_IDS[u.dtype], c, s, groups
    d.n, d.l = u.shape[0], u.shape[1] if u.dim() == 3 else 1
    pad = (lambda t: t.stride()) if u.dim() == 3 else (lambda t: (t.stride(0), 0, *t.stride()[1:]))
    _set(d.u_strides, pad(u))
    _set(d.delta_strides, pad(delta))
    if z is not None:
        _set(d.z_strides, pad(z))
    _set(d.b_strides, pad(B))
    _set(d.c_strides, pad(C))
    return d, A.contiguous(), B, C, _dense(D), _dense(delta_bias)


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
                   delta_softplus: bool = False, initial_state: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, return_final_state: bool = False):
    """The scan ``h[t] = exp(dt A) h[t-1] + dt u[t] B[t]``, ``y[t] = (sum_s C[t] h[t] + D u[t]) silu(z[t])`` over ``u``
    [N, L, C] with ``dt = delta + delta_bias`` (``softplus`` of it if asked).

    ``A`` [C, S], ``D`` and ``delta_bias`` [C] are float32; ``B`` and ``C`` [N, L, S], or [N, L, groups, S] where each group of
    channels has its own.  ``initial_state`` and the returned state are float32 [N, C, S]."""
    what = "selective_scan"
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.selective_scan(u, delta, A, B, C, D, z, delta_bias, bool(delta_softplus), initial_state, lengths,
                                bool(return_final_state))
        if y is not None:
            return answered(y)
    _check_input(what, "u", u, 3)
    d, A, B, C, D, delta_bias = _check_scan(what, u, delta, A, B, C, D, z, delta_bias)
    n, length, c = u.shape
    _check_like(what, "initial_state", initial_state, (n, c, d.s), torch.float32, u.device)
    _check_like(what, "lengths", lengths, (n,), torch.int32, u.device)
    refuse_grad(what, u, delta, A, B, C, D, z, delta_bias, initial_state)
    initial_state, lengths = _dense(initial_state), _dense(lengths)
    d.delta_softplus = int(bool(delta_softplus))
    y = torch.empty((n, length, c), dtype=u.dtype, device=u.device)
    _set(d.y_strides, y.stride())
    final = torch.empty((n, c, d.s), dtype=torch.float32, device=u.device) if return_final_state else None
    lib = nat.load()
    nbytes = ctypes.c_int64()
    with torch.cuda.device(u.device):
        nat.check(lib.fdnn_selective_scan_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
        ws = workspace(nbytes.value, u.device)
        nat.check(lib.fdnn_selective_scan_fwd(
            ctypes.byref(d), u.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), address(D), address(z),
            address(delta_bias), address(initial_state), address(lengths), y.data_ptr(), address(final), address(ws), nbytes.value,
            torch.cuda.current_stream().cuda_stream))
    return (y, final) if return_final_state else y


def selective_scan_step(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                        slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``selective_scan`` of the next token of each row: ``u``, ``delta``, ``z`` [N, C], ``B`` and ``C`` [N, S] or
    [N, groups, S]; ``state`` [slots, C, S] float32 is updated in place."""
    what = "selective_scan_step"
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.selective_scan_step(u, delta, A, B, C, state, D, z, delta_bias, bool(delta_softplus), slots)
        if y is not None:
            return answered(y)
    _check_input(what, "u", u, 2)
    d, A, B, C, D, delta_bias = _check_scan(what, u, delta, A, B, C, D, z, delta_bias)
    n, c = u.shape
    _check_cache(what, "state", state, (c, d.s), torch.float32, u, slots)
    refuse_grad(what, u, delta, A, B, C, D, z, delta_bias, state)
    slots = _dense(slots)
    d.delta_softplus = int(bool(delta_softplus))
    y = torch.empty((n, c), dtype=u.dtype, device=u.device)
    _set(d.y_strides, (c, 0, 1))
    with torch.cuda.device(u.device):
        nat.check(nat.load().fdnn_selective_scan_step(
            ctypes.byref(d), u.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), address(D), address(z),
            address(delta_bias), state.data_ptr(), state.shape[0], address(slots), y.data_ptr(),
            torch.cuda.current_stream().cuda_stream))
    increment_version(state)
    return y
