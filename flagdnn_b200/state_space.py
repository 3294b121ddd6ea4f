"""A state space mixer: the block of a sequence model whose tokens meet through a selective scan instead of attention.

    x -> mm (in) -> causal_conv1d (silu) -> mm (delta, B, C) -> selective_scan (gated) -> group_norm per token -> mm (out)

Prompts run through :meth:`StateSpaceMixer.forward`, which returns the state behind them; the next tokens through
:meth:`StateSpaceMixer.step`, which continues states in place, each row at its slot of a cache. Everything is computed by this
library's kernels; what the products leave is read in place (delta, B and C are columns of one product's result).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import conv_host, norm_host, sequence_host


@dataclass
class MixerState:
    """What a row carries from token to token: the convolution's last inputs and the scan's states."""
    conv: torch.Tensor    # [slots, width - 1, inner]
    scan: torch.Tensor    # [slots, inner, states] float32

    def put(self, slots: torch.Tensor, other: "MixerState") -> None:
        """Row n of ``other`` (or its only one) into slot ``slots[n]``, as after the prompts that begin there; a slot outside the
        cache marks an idle row, which is not written."""
        n = slots.numel()
        if slots.dim() != 1 or any(t.shape[0] not in (n, 1) for t in (other.conv, other.scan)):
            raise RuntimeError(f"put: {tuple(slots.shape)} slots for {other.conv.shape[0]} and {other.scan.shape[0]} rows")
        if self.conv.shape[0] != self.scan.shape[0]:
            raise RuntimeError(f"put: a cache of {self.conv.shape[0]} and {self.scan.shape[0]} slots")
        if n == 0 or self.conv.shape[0] == 0:
            return
        slots = slots.to(self.conv.device)
        conv, scan = (t.expand(n, *t.shape[1:]) for t in (other.conv, other.scan))
        # an idle row writes once more what the first other one does (or what slot 0 has, where all are idle): the host need not
        # know which rows those are
        live = (slots >= 0) & (slots < self.conv.shape[0])
        first, any_live = live.to(torch.uint8).argmax(), live.any()
        rows = torch.where(live, torch.arange(n, device=slots.device), first)
        at = torch.where(any_live, slots[rows], 0).long()
        self.conv[at] = torch.where(any_live, conv[rows], self.conv[at])
        self.scan[at] = torch.where(any_live, scan[rows], self.scan[at])


class StateSpaceMixer:
    """Random-init parameters; ``model`` channels in and out, ``inner`` channels in the scan."""

    def __init__(self, model: int, inner: int, states: int = 16, rank: int = 32, width: int = 4, norm_groups: int = 8,
                 device="cuda", dtype: torch.dtype = torch.bfloat16, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        self.model, self.inner, self.states, self.rank, self.width, self.norm_groups = model, inner, states, rank, width, norm_groups
        self.device, self.dtype = torch.device(device), dtype

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g) * rows ** -0.5).to(dtype).to(device)

        self.w_in = weight(model, 2 * inner)
        self.w_out = weight(inner, model)
        self.w_steps = weight(inner, rank + 2 * states)
        self.w_delta = weight(rank, inner)
        self.w_conv = (torch.randn(inner, width, generator=g) * width ** -0.5).to(dtype).to(device)
        self.b_conv = (torch.randn(inner, generator=g) * 0.1).to(dtype).to(device)
        self.A = -torch.arange(1, states + 1).float().repeat(inner, 1).to(device)
        self.D = torch.ones(inner, device=device)
        dt = torch.exp(torch.rand(inner, generator=g) * 4.6 - 6.9)             # steps of 0.001 .. 0.1
        self.delta_bias = (dt + torch.log(-torch.expm1(-dt))).to(device)
        self.w_norm = torch.ones(inner, dtype=dtype, device=device)
        self.b_norm = torch.zeros(inner, dtype=dtype, device=device)

    def new_state(self, slots: int) -> MixerState:
        return MixerState(torch.zeros(slots, self.width - 1, self.inner, dtype=self.dtype, device=self.device),
                          torch.zeros(slots, self.inner, self.states, device=self.device))

    def _steps(self, v: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """delta [T, inner], B and C [T, states] of tokens v [T, inner]."""
        steps = conv_host.mm(v, self.w_steps)
        delta = conv_host.mm(steps[:, :self.rank], self.w_delta)
        return delta, steps[:, self.rank:self.rank + self.states], steps[:, self.rank + self.states:]

    def _out(self, y: torch.Tensor) -> torch.Tensor:
        return conv_host.mm(norm_host.group_norm(y, self.norm_groups, self.w_norm, self.b_norm), self.w_out)

    @torch.no_grad()
    def forward(self, x: torch.Tensor, state: Optional[MixerState] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, MixerState]:
        """Prompts x [N, L, model], behind ``state`` if given (row n at slot n of N slots or more), ragged by ``lengths``: the
        outputs (of padding tokens: those of a zero) and the state behind each row."""
        n, length, _ = x.shape
        if state is not None:
            state = MixerState(state.conv[:n], state.scan[:n])
        both = conv_host.mm(x.reshape(n * length, self.model), self.w_in).view(n, length, 2 * self.inner)
        v, conv_state = sequence_host.causal_conv1d(both[..., :self.inner], self.w_conv, self.b_conv, "silu",
                                                    None if state is None else state.conv, lengths, True)
        delta, B, C = self._steps(v.view(n * length, self.inner))
        y, scan_state = sequence_host.selective_scan(
            v, delta.view(n, length, self.inner), self.A, B.unflatten(0, (n, length)), C.unflatten(0, (n, length)), self.D,
            both[..., self.inner:], self.delta_bias, True, None if state is None else state.scan, lengths, True)
        out = self._out(y.view(n * length, self.inner))
        return out.view(n, length, self.model), MixerState(conv_state, scan_state)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: MixerState, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The next token of each row, x [N, model]; row n continues slot ``slots[n]`` (default n) of ``state`` in place."""
        both = conv_host.mm(x, self.w_in)
        v = sequence_host.causal_conv1d_step(both[:, :self.inner], state.conv, self.w_conv, self.b_conv, "silu", slots)
        delta, B, C = self._steps(v)
        y = sequence_host.selective_scan_step(v, delta, self.A, B, C, state.scan, self.D, both[:, self.inner:], self.delta_bias, True,
                                              slots)
        return self._out(y)
