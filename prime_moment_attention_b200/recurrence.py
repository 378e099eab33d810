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

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DT, _require_cuda, _stream, check_faults


def _blc(t: Optional[torch.Tensor]):
    """pma_seq_tensor of a [B, L, C] (or [N, C]) tensor whose last axis is contiguous; None stays None."""
    if t is None:
        return None
    sb, sl = (t.stride(0), t.stride(1)) if t.dim() == 3 else (t.stride(0), 0)
    return ctypes.byref(_lib.SeqTensor(t.data_ptr(), _DT[t.dtype], sb, 0, sl))


def _rows_ok(t: torch.Tensor) -> torch.Tensor:
    """`t`, copied only where the kernels cannot address it: the channel axis must be contiguous."""
    t = t.detach()
    if t.shape[-1] > 1 and t.stride(-1) != 1 or any(s < 0 for s in t.stride()):
        t = t.contiguous()
    return t


def _like(name: str, t, shape, dtype, dev) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != dev:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on {dev}")
    return t


def _check(x, f, bias, gate, dims: int):
    dev = _require_cuda(x, f)
    if x.dim() != dims:
        raise ValueError(f"x must have {dims} axes; got shape {tuple(x.shape)}")
    if x.dtype not in _DT:
        raise TypeError(f"unsupported dtype {x.dtype}: float32 or bfloat16")
    if x.shape[-1] == 0:
        raise ValueError("x must have at least one channel")
    _like("f", f, x.shape, x.dtype, dev)
    if gate is not None:
        _like("gate", gate, x.shape, x.dtype, dev)
    if bias is not None:
        _like("bias", bias, x.shape[-1:], torch.float32, dev)
    return dev


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, bias, gate, h0, reset):
        B, L, C = x.shape
        dev = x.device
        lib = _lib.load()
        xs, fs = _rows_ok(x), _rows_ok(f)
        gs = _rows_ok(gate) if gate is not None else None
        bs = bias.detach().contiguous() if bias is not None else None
        hs = h0.detach().contiguous() if h0 is not None else None
        y = torch.empty(B, L, C, dtype=x.dtype, device=dev)
        h = torch.empty(B, C, dtype=torch.float32, device=dev)
        n = lib.pma_gated_scan_workspace_bytes(B, L, C)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.check("pma_gated_scan", lib.pma_gated_scan(
            B, L, C, _blc(xs), _blc(fs), _blc(gs), _ptr(bs), _ptr(hs), _ptr(reset), _blc(y), h.data_ptr(),
            ws.data_ptr() if n else None, n, _stream(dev)))
        ctx.save_for_backward(xs, fs, gs, bs, hs, reset, ws)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        xs, fs, gs, bs, hs, reset, ws = ctx.saved_tensors
        B, L, C = xs.shape
        dev = xs.device
        lib = _lib.load()
        check_faults("gated_scan backward")
        dy = _rows_ok(dy) if dy is not None else torch.zeros(1, 1, C, dtype=xs.dtype, device=dev).expand(B, L, C)
        dh = dh.detach().contiguous() if dh is not None else None
        new = lambda: torch.empty(B, L, C, dtype=xs.dtype, device=dev)  # noqa: E731
        dx, df = new(), new()
        dg = new() if gs is not None else None
        db = torch.empty(C, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        d0 = torch.empty(B, C, dtype=torch.float32, device=dev) if ctx.needs_input_grad[4] else None
        n = lib.pma_gated_scan_backward_workspace_bytes(B, L, C)
        w2 = torch.empty(max(n, 1), dtype=torch.uint8, device=dev)
        _lib.check("pma_gated_scan_backward", lib.pma_gated_scan_backward(
            B, L, C, _blc(xs), _blc(fs), _blc(gs), _ptr(bs), _ptr(hs), _ptr(reset), _blc(dy), _ptr(dh), _blc(dx),
            _blc(df), _blc(dg), _ptr(db), _ptr(d0), ws.data_ptr() if ws.numel() else None, ws.numel(), w2.data_ptr(),
            n, _stream(dev)))
        return dx, df, db, dg, d0, None


def gated_scan(x: torch.Tensor, f: torch.Tensor, bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
               reset: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence over x, f (and gate) [B, L, C], bf16 or float32, with any strides on B and L.

    bias [C] and h0 [B, C] are float32; reset [B, L] (bool or uint8) cuts the state before a token.
    Returns (y [B, L, C] in x's dtype, h_L [B, C] float32).  Differentiable; the backward pass reads
    x, f, gate and one float32 state per channel and 128 tokens.  Gradients repeat bit for bit."""
    dev = _check(x, f, bias, gate, 3)
    check_faults("gated_scan")
    B, L, C = x.shape
    if h0 is not None:
        _like("h0", h0, (B, C), torch.float32, dev)
    if reset is not None:
        if not isinstance(reset, torch.Tensor) or reset.dtype not in (torch.bool, torch.uint8):
            raise TypeError("reset must be a bool or uint8 tensor")
        reset = _like("reset", reset, (B, L), reset.dtype, dev).contiguous()
    return _Scan.apply(x, f, bias, gate, h0, reset)


def gated_scan_step(x: torch.Tensor, f: torch.Tensor, h: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    gate: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                    inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token: x, f (and gate) [N, C] and the float32 state h [N, C]; returns (y, new h).

    With inplace=True h itself is updated.  With `rows` (int32 [N], distinct) h is a pool [P, C] and
    batch row n advances pool row rows[n] in place; rows outside the pool are skipped (y = 0)."""
    dev = _check(x, f, bias, gate, 2)
    N, C = x.shape
    if rows is not None:
        inplace = True
        rows = _like("rows", rows, (N,), torch.int32, dev).contiguous()
        _like("h", h, (h.shape[0], C) if isinstance(h, torch.Tensor) and h.dim() == 2 else (N, C), torch.float32, dev)
    else:
        _like("h", h, (N, C), torch.float32, dev)
    if inplace and not h.is_contiguous():
        raise ValueError("h must be contiguous to be updated in place")
    h = h.detach().contiguous()
    out = h if inplace else torch.empty_like(h)
    xs, fs = _rows_ok(x), _rows_ok(f)
    gs = _rows_ok(gate) if gate is not None else None
    y = torch.empty(N, C, dtype=x.dtype, device=dev)
    _lib.check("pma_gated_scan_step", _lib.load().pma_gated_scan_step(
        N, C, _blc(xs), _blc(fs), _blc(gs), _ptr(bias.detach().contiguous()) if bias is not None else None,
        h.data_ptr(), out.data_ptr(), _ptr(rows), h.shape[0], _blc(y), _stream(dev)))
    return y, out
