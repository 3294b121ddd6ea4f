"""Group norm, its gradient, the causal convolution and the selective scan from their definitions, in 64 bits on the CPU.

Test infrastructure.  Inputs may be of any type and on any device; results are float64 on the CPU.  Loops over rows and
tokens where the definition has them.
"""
from __future__ import annotations

import math

import torch


def _64(t):
    return None if t is None else t.detach().double().cpu()


def activate(v: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.relu(v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    assert act == "none"
    return v


def slope(v: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return (v > 0).double()
    if act == "silu":
        p = torch.sigmoid(v)
        return p + v * p * (1 - p)
    if act == "gelu":
        return torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (v + 0.044715 * v ** 3))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)
    return torch.ones_like(v)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, act="none"):
    """(y, mean, rstd)"""
    x = _64(x)
    n, c = x.shape[:2]
    rows = x.reshape(n, groups, -1)
    mean = rows.mean(2)
    rstd = 1 / torch.sqrt(((rows - mean[..., None]) ** 2).mean(2) + eps)
    xh = ((rows - mean[..., None]) * rstd[..., None]).reshape(n, c, -1)
    w = torch.ones(c, dtype=torch.float64) if weight is None else _64(weight)
    b = torch.zeros(c, dtype=torch.float64) if bias is None else _64(bias)
    return activate(xh * w[:, None] + b[:, None], act).reshape(x.shape), mean, rstd


def group_norm_grad(dy, x, groups, weight=None, bias=None, eps=1e-5, act="none"):
    """(dx, dweight, dbias) by the formulas"""
    x, dy = _64(x), _64(dy)
    n, c = x.shape[:2]
    _, mean, rstd = group_norm(x, groups, eps=eps)
    xh = ((x.reshape(n, groups, -1) - mean[..., None]) * rstd[..., None]).reshape(n, c, -1)
    w = torch.ones(c, dtype=torch.float64) if weight is None else _64(weight)
    b = torch.zeros(c, dtype=torch.float64) if bias is None else _64(bias)
    g = dy.reshape(n, c, -1) * slope(xh * w[:, None] + b[:, None], act)
    dw, db = (g * xh).sum((0, 2)), g.sum((0, 2))
    gw, xg = (g * w[:, None]).reshape(n, groups, -1), xh.reshape(n, groups, -1)
    dx = rstd[..., None] * (gw - gw.mean(2, keepdim=True) - xg * (gw * xg).mean(2, keepdim=True))
    return dx.reshape(x.shape), dw, db


def causal_conv1d(x, weight, bias=None, act="none", initial=None, lengths=None):
    """(y, final state)"""
    x, w, b, initial = _64(x), _64(weight), _64(bias), _64(initial)
    n, length, c = x.shape
    width = w.shape[1]
    y, final = torch.zeros_like(x), torch.zeros(n, width - 1, c, dtype=torch.float64)
    for i in range(n):
        end = length if lengths is None else int(lengths[i])
        before = torch.zeros(width - 1, c, dtype=torch.float64) if initial is None else initial[i]
        xs = torch.cat([before, x[i, :end]])
        for t in range(end):
            v = (xs[t:t + width] * w.t()).sum(0)
            y[i, t] = activate(v if b is None else v + b, act)
        final[i] = xs[end:end + width - 1]
    return y, final


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, initial=None, lengths=None):
    """(y, final state); B and C [N, L, groups, S]"""
    u, delta, A, B, C, D, z, delta_bias, initial = (_64(t) for t in (u, delta, A, B, C, D, z, delta_bias, initial))
    n, length, c = u.shape
    s, per = A.shape[1], c // B.shape[2]
    dt = delta if delta_bias is None else delta + delta_bias
    if softplus:
        dt = dt.clamp_min(0) + torch.log1p(torch.exp(-dt.abs()))
    y, final = torch.zeros_like(u), torch.zeros(n, c, s, dtype=torch.float64)
    for i in range(n):
        end = length if lengths is None else int(lengths[i])
        h = torch.zeros(c, s, dtype=torch.float64) if initial is None else initial[i].clone()
        for t in range(end):
            d = dt[i, t][:, None]
            h = torch.exp(d * A) * h + d * u[i, t][:, None] * B[i, t].repeat_interleave(per, 0)
            v = (h * C[i, t].repeat_interleave(per, 0)).sum(1)
            if D is not None:
                v = v + D * u[i, t]
            y[i, t] = v if z is None else v * z[i, t] * torch.sigmoid(z[i, t])
        final[i] = h
    return y, final
