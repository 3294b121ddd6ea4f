"""The gated delta rule and a product with its epilogue from their definitions, in 64 bits on the CPU.

Test infrastructure.  Inputs may be of any type and on any device; results are float64 on the CPU.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .sequence_oracle import _64, activate


class Rule(NamedTuple):
    y: torch.Tensor
    state: torch.Tensor
    y_size: torch.Tensor        # sums of the sizes of the terms that y and the state are made of, for tolerances
    state_size: torch.Tensor


def gated_delta_rule(q, k, v, delta, beta, A=None, delta_bias=None, delta_softplus=False, beta_sigmoid=False, qk_norm=False, scale=None,
                     initial_state=None, lengths: Optional[list] = None) -> Rule:
    """Token by token over [N, L, heads, channels]; tokens from lengths[n] on are not read."""
    q, k, v, delta, beta, A, delta_bias, initial_state = (_64(t) for t in (q, k, v, delta, beta, A, delta_bias, initial_state))
    n, length, heads, dv = v.shape
    dk = q.shape[-1]
    scale = dk ** -0.5 if scale is None else scale
    state = torch.zeros(n, heads, dv, dk, dtype=torch.float64) if initial_state is None else initial_state.clone()
    size = state.abs()
    y, y_size = torch.zeros_like(v), torch.zeros_like(v)
    for i in range(n):
        for t in range(length if lengths is None else lengths[i]):
            kt, qt = k[i, t], q[i, t]
            if qk_norm:
                kt, qt = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (kt, qt))
            kt, qt = (x.repeat_interleave(heads // x.shape[0], 0) for x in (kt, qt * scale))
            dt = delta[i, t] if delta_bias is None else delta[i, t] + delta_bias
            dt = torch.log1p(torch.exp(-dt.abs())) + dt.clamp_min(0) if delta_softplus else dt
            a = torch.exp(dt if A is None else A * dt)[:, None, None]
            b = (1 / (1 + torch.exp(-beta[i, t])) if beta_sigmoid else beta[i, t])[:, None]
            old = a * state[i]
            u = b * (v[i, t] - (old * kt[:, None]).sum(-1))
            u_size = b.abs() * (v[i, t].abs() + (old * kt[:, None]).abs().sum(-1))
            state[i] = old + u[..., None] * kt[:, None]
            size[i] = a * size[i] + u_size[..., None] * kt[:, None].abs()
            y[i, t] = (state[i] * qt[:, None]).sum(-1)
            y_size[i, t] = (size[i] * qt[:, None].abs()).sum(-1)
    return Rule(y, state, y_size, size)


def mm_bias_act(a, b, bias=None, residual=None, activation="none"):
    y = _64(a) @ _64(b)
    for t in (bias, residual):
        if t is not None:
            y = y + _64(t)
    return activate(y, activation)
