"""A gated linear recurrence per channel, for training, prefill and single tokens.

    a_t = sigmoid(f_t + bias)      h_t = a_t h_{t-1} + (1 - a_t) x_t      y_t = h_t silu(gate_t)

over [B, L, C] (y = h without a gate), on pma_gated_scan, its gradient and its one-token step
(include/pma.h).  Where the moment attention keeps a D x D state per head, this keeps one number
per channel: a cheap mixer to put beside it.  Unlike the attention entries this one trains:
gated_scan is differentiable in x, f, bias, gate and h0.

    y, h = gated_scan(x, f, bias, gate, h0, reset)            # prefill or training; h continues it
    y, h = gated_scan_step(x1, f1, h, bias=bias, gate=gate1)  # one token

GatedRecurrence is the layer around it, with the interface of the attention modules.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import torch_ops
from .ops import _require_cuda, check_faults

_fns = None
_c = None


def _ops():
    """The operators (loaded once): gated_scan, gated_scan_step, gated_scan_step_."""
    global _fns
    if _fns is None:
        torch_ops.load()
        n = torch.ops.pma
        _fns = (n.gated_scan.default, n.gated_scan_step.default, n.gated_scan_step_.default)
    return _fns


def _direct():
    global _c
    if _c is None:
        _c = torch_ops.direct()
    return _c


def gated_scan(x: torch.Tensor, f: torch.Tensor, bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
               reset: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence over x, f (and gate) [B, L, C], bf16 or float32, with any strides on B and L.

    bias [C] and h0 [B, C] are float32; reset [B, L] (bool or uint8) cuts the state before a token.
    Returns (y [B, L, C] in x's dtype, h_L [B, C] float32).  Differentiable; the backward pass reads
    x, f, gate and one float32 state per channel and 128 tokens.  Gradients repeat bit for bit."""
    if not torch.compiler.is_compiling():
        if getattr(x, "is_cuda", False):
            check_faults("gated_scan")
        r = _direct().gated_scan(x, f, bias, gate, h0, reset)
        if r is not NotImplemented:
            return r
    _require_cuda(x, f)
    torch_ops.watch_faults()
    return _ops()[0](x, f, bias, gate, h0, reset)


def gated_scan_step(x: torch.Tensor, f: torch.Tensor, h: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    gate: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                    inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token: x, f (and gate) [N, C] and the float32 state h [N, C]; returns (y, new h).

    With inplace=True h itself is updated.  With `rows` (int32 [N], distinct) h is a pool [P, C] and
    batch row n advances pool row rows[n] in place; rows outside the pool are skipped (y = 0).
    Inference only."""
    pool = rows is not None or inplace
    if not torch.compiler.is_compiling():
        c = _direct()
        r = c.gated_scan_step_(x, f, h, bias, gate, rows) if pool else c.gated_scan_step(x, f, h, bias, gate)
        if r is not NotImplemented:
            return (r, h) if pool else r
    _require_cuda(x, f, h)
    if pool:
        return _ops()[2](x, f, h, bias, gate, rows), h
    return _ops()[1](x, f, h, bias, gate)


class GatedRecurrence(nn.Module):
    """Sequence mixer on the gated recurrence, in the place of an attention module: one projection to
    (x, f, gate), the scan over `width` channels, one projection back.  Trains (the attention modules
    do not); prefill and decode carry the state (h [B, width] float32,).  The decays start spread
    over [min_decay, max_decay], evenly in their time constants' logarithm."""

    def __init__(self, hidden_size: int, width: Optional[int] = None, min_decay: float = 0.9,
                 max_decay: float = 0.9999):
        super().__init__()
        if not 0.0 < min_decay <= max_decay < 1.0:
            raise ValueError("decays must satisfy 0 < min_decay <= max_decay < 1")
        self.hidden_size = hidden_size
        self.width = width or hidden_size
        self.in_proj = nn.Linear(hidden_size, 3 * self.width, bias=False)
        self.o_proj = nn.Linear(self.width, hidden_size, bias=False)
        lo, hi = math.log(1.0 - min_decay), math.log(1.0 - max_decay)
        z = torch.exp(torch.linspace(lo, hi, self.width))  # 1 - decay
        self.decay_bias = nn.Parameter(torch.log((1.0 - z) / z))

    def forward(self, hidden_states: torch.Tensor, state: Optional[Tuple[torch.Tensor, ...]] = None,
                return_state: bool = False, reset: Optional[torch.Tensor] = None):
        """hidden_states [B, L, hidden]; state (h,) of the tokens before; reset [B, L] marks the first
        tokens of packed documents.  Returns (output, (h,) or None)."""
        x, f, gate = self.in_proj(hidden_states).split(self.width, dim=-1)
        h0 = state[0] if state is not None else None
        bias = self.decay_bias.float()
        if hidden_states.shape[1] == 1 and reset is None and not torch.is_grad_enabled():
            if h0 is None:
                h0 = torch.zeros(x.shape[0], self.width, dtype=torch.float32, device=x.device)
            y, h = gated_scan_step(x[:, 0], f[:, 0], h0, bias=bias, gate=gate[:, 0])
            y = y[:, None]
        else:
            y, h = gated_scan(x, f, bias, gate, h0, reset)
        return self.o_proj(y), ((h,) if return_state else None)

    def step_(self, xfg: torch.Tensor, state: Tuple[torch.Tensor, ...]) -> torch.Tensor:
        """One token from its projections [B, 3 width] with the state updated in place; before o_proj."""
        x, f, gate = xfg.split(self.width, dim=-1)
        return gated_scan_step(x, f, state[0], bias=self.decay_bias.float(), gate=gate, inplace=True)[0]
