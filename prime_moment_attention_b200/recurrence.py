"""A gated linear recurrence per channel, for training, prefill and single tokens.

    a_t = sigmoid(f_t + bias)      h_t = a_t h_{t-1} + (1 - a_t) x_t      y_t = h_t silu(gate_t)

over [B, L, C] (y = h without a gate), on pma_gated_scan, its gradient and its one-token step
(include/pma.h).  Where the moment attention keeps a D x D state per head, this keeps one number
per channel: a cheap mixer to put beside it.  Unlike the attention entries this one trains:
gated_scan is differentiable in x, f, bias, gate and h0.

    y, h = gated_scan(x, f, bias, gate, h0, reset)            # prefill or training; h continues it
    y, h = gated_scan_step(x1, f1, h, bias=bias, gate=gate1)  # one token
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import torch_ops
from .ops import _require_cuda, check_faults

_fns = None


def _ops():
    """The operators (loaded once): gated_scan, gated_scan_step, gated_scan_step_."""
    global _fns
    if _fns is None:
        torch_ops.load()
        n = torch.ops.pma
        _fns = (n.gated_scan.default, n.gated_scan_step.default, n.gated_scan_step_.default)
    return _fns


def gated_scan(x: torch.Tensor, f: torch.Tensor, bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
               reset: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence over x, f (and gate) [B, L, C], bf16 or float32, with any strides on B and L.

    bias [C] and h0 [B, C] are float32; reset [B, L] (bool or uint8) cuts the state before a token.
    Returns (y [B, L, C] in x's dtype, h_L [B, C] float32).  Differentiable; the backward pass reads
    x, f, gate and one float32 state per channel and 128 tokens.  Gradients repeat bit for bit."""
    _require_cuda(x, f)
    check_faults("gated_scan")
    return _ops()[0](x, f, bias, gate, h0, reset)


def gated_scan_step(x: torch.Tensor, f: torch.Tensor, h: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    gate: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                    inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token: x, f (and gate) [N, C] and the float32 state h [N, C]; returns (y, new h).

    With inplace=True h itself is updated.  With `rows` (int32 [N], distinct) h is a pool [P, C] and
    batch row n advances pool row rows[n] in place; rows outside the pool are skipped (y = 0).
    Inference only."""
    _require_cuda(x, f, h)
    if rows is not None or inplace:
        return _ops()[2](x, f, h, bias, gate, rows), h
    return _ops()[1](x, f, h, bias, gate)
