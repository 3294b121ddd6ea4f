"""Host side of the gated delta rule, over prompts and for single tokens.

Tensors are laid out as for the state space operators beside it: ``[N, L, heads, channels]``, tokens in order (any strides are
taken; columns of a wider projection need no copy), ``lengths`` (int32 [N]) for ragged batches, whose tokens from ``lengths[n]`` on
are never read and give zeros.  A head's state is float32 ``[value channels, key channels]``: ``[N, heads, V, K]``, the caller's; the
step function updates a cache of states in place, at ``slots`` (int32 [N]; a slot outside the cache marks an idle row, whose
output is zero; two rows must not share one), and it counts as written for autograd's check of saved tensors.  These are
operators of the forward pass: tensors that ask for a gradient, or carry a tangent, are refused.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _native as nat
from . import conv_host as _conv
from .norm_host import _DTYPE_IDS, address, answered, refuse_grad, workspace
from .sequence_host import _check_cache, _check_input, _check_like, _dense, _set

MAX_KEY, MAX_VALUE, MAX_HEADS = 256, 1024, 65535


def _check_rule(what: str, q, k, v, delta, beta, A, delta_bias, delta_softplus, beta_sigmoid, qk_norm, scale):
    """The descriptor for these tensors, and A and delta_bias as the library takes them."""
    rows, heads, dv = tuple(v.shape[:-2]), v.shape[-2], v.shape[-1]
    if q.dim() != v.dim() or tuple(q.shape[:-2]) != rows:
        raise RuntimeError(f"{what}: q must have shape {(*rows, 'key heads', 'key channels')}, got {tuple(q.shape)}")
    key_heads, dk = q.shape[-2:]
    if key_heads < 1 or heads % key_heads != 0:
        raise RuntimeError(f"{what}: {heads} heads cannot share {key_heads} key heads evenly")
    if not 1 <= dk <= MAX_KEY or not 1 <= dv <= MAX_VALUE or heads > MAX_HEADS:
        raise NotImplementedError(f"flag_dnn {what} takes keys of 1 to {MAX_KEY} channels, values of 1 to {MAX_VALUE} and at most "
                                  f"{MAX_HEADS} heads, got {dk}, {dv} and {heads}")
    _check_like(what, "q", q, q.shape, v.dtype, v.device)
    _check_like(what, "k", k, q.shape, v.dtype, v.device)
    if delta.dtype not in (v.dtype, torch.float32):
        raise RuntimeError(f"{what}: delta must be {v.dtype} or torch.float32, got {delta.dtype}")
    for name, t in (("delta", delta), ("beta", beta)):
        _check_like(what, name, t, (*rows, heads), delta.dtype, v.device)
    for name, t in (("A", A), ("delta_bias", delta_bias)):
        _check_like(what, name, t, (heads,), torch.float32, v.device)
    d = nat.DeltaRuleDesc()
    d.dtype, d.gate_dtype, d.key_heads, d.heads, d.dk, d.dv = _DTYPE_IDS[v.dtype], _DTYPE_IDS[delta.dtype], key_heads, heads, dk, dv
    d.n, d.l = v.shape[0], v.shape[1] if v.dim() == 4 else 1
    d.delta_softplus, d.beta_sigmoid, d.qk_norm = int(bool(delta_softplus)), int(bool(beta_sigmoid)), int(bool(qk_norm))
    d.scale = dk ** -0.5 if scale is None else float(scale)
    pad = (lambda t: t.stride()) if v.dim() == 4 else (lambda t: (t.stride(0), 0, *t.stride()[1:]))
    for field, t in ((d.q_strides, q), (d.k_strides, k), (d.v_strides, v), (d.delta_strides, delta), (d.beta_strides, beta)):
        _set(field, pad(t))
    return d, _dense(A), _dense(delta_bias)


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, delta: torch.Tensor, beta: torch.Tensor,
                     A: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                     beta_sigmoid: bool = False, qk_norm: bool = False, scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                     return_final_state: bool = False):
    """``S <- a S``, ``S <- S + b (v - S k) k^T``, ``y = S q * scale`` over the tokens of ``v`` [N, L, H, V], with the decay
    ``a = exp(A dt)`` (``exp(dt)`` without ``A``), ``dt = delta + delta_bias`` (``softplus`` of it if asked) and ``b = beta`` (``sigmoid``
    of it if asked).

    ``q`` and ``k`` [N, L, G, K]: each key head serves ``H / G`` neighbouring heads; with ``qk_norm`` they are divided by
    ``sqrt(sum of squares + 1e-6)``.  ``delta`` and ``beta`` [N, L, H] are of ``v``'s type or float32, ``A`` and ``delta_bias`` [H]
    float32; ``scale`` is ``K ** -0.5`` if None.  ``initial_state`` and the returned state are float32 [N, H, V, K].
    Prompts are taken in chunks of 64 tokens: an input that is not finite can make its whole chunk not finite, and what a token
    brings to a value channel is held to 2^-22 of itself or 2^-39 of the most that one of its chunk does. Long rows are cut into
    segments where few rows and heads run: a row's last bits can depend on its batch. Decays above one are taken as long as their
    product is at most 2^18 over any stretch of a chunk (past that the chunk and what follows are NaN) and an fp32 number over any
    stretch of the row, also where the state stays small or zero."""
    what = "gated_delta_rule"
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.gated_delta_rule(q, k, v, delta, beta, A, delta_bias, bool(delta_softplus), bool(beta_sigmoid), bool(qk_norm), scale,
                                  initial_state, lengths, bool(return_final_state))
        if y is not None:
            return answered(y)
    _check_input(what, "v", v, 4)
    d, A, delta_bias = _check_rule(what, q, k, v, delta, beta, A, delta_bias, delta_softplus, beta_sigmoid, qk_norm, scale)
    _check_like(what, "initial_state", initial_state, (d.n, d.heads, d.dv, d.dk), torch.float32, v.device)
    _check_like(what, "lengths", lengths, (d.n,), torch.int32, v.device)
    refuse_grad(what, q, k, v, delta, beta, A, delta_bias, initial_state)
    initial_state, lengths = _dense(initial_state), _dense(lengths)
    y = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    _set(d.y_strides, y.stride())
    final = torch.empty((d.n, d.heads, d.dv, d.dk), dtype=torch.float32, device=v.device) if return_final_state else None
    lib = nat.load()
    nbytes = ctypes.c_int64()
    with torch.cuda.device(v.device):
        nat.check(lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
        ws = workspace(nbytes.value, v.device)
        nat.check(lib.fdnn_gated_delta_rule_fwd(
            ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), delta.data_ptr(), beta.data_ptr(), address(A), address(delta_bias),
            address(initial_state), address(lengths), y.data_ptr(), address(final), address(ws), nbytes.value,
            torch.cuda.current_stream().cuda_stream))
    return (y, final) if return_final_state else y


def gated_delta_rule_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, delta: torch.Tensor, beta: torch.Tensor,
                          state: torch.Tensor, A: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
                          delta_softplus: bool = False, beta_sigmoid: bool = False, qk_norm: bool = False,
                          scale: Optional[float] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gated_delta_rule`` of the next token of each row: ``q`` and ``k`` [N, G, K], ``v`` [N, H, V], ``delta`` and ``beta`` [N, H];
    ``state`` [slots, H, V, K] float32 is updated in place."""
    what = "gated_delta_rule_step"
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.gated_delta_rule_step(q, k, v, delta, beta, state, A, delta_bias, bool(delta_softplus), bool(beta_sigmoid),
                                       bool(qk_norm), scale, slots)
        if y is not None:
            return answered(y)
    _check_input(what, "v", v, 3)
    d, A, delta_bias = _check_rule(what, q, k, v, delta, beta, A, delta_bias, delta_softplus, beta_sigmoid, qk_norm, scale)
    _check_cache(what, "state", state, (d.heads, d.dv, d.dk), torch.float32, v, slots)
    refuse_grad(what, q, k, v, delta, beta, state, A, delta_bias)
    slots = _dense(slots)
    y = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    _set(d.y_strides, (y.stride(0), 0, *y.stride()[1:]))
    with torch.cuda.device(v.device):
        nat.check(nat.load().fdnn_gated_delta_rule_step(
            ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), delta.data_ptr(), beta.data_ptr(), address(A), address(delta_bias),
            state.data_ptr(), state.shape[0], address(slots), y.data_ptr(), torch.cuda.current_stream().cuda_stream))
    increment_version(state)
    return y
