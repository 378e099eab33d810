"""torch.ops.pma: the prefill and decode step as PyTorch operators (csrc/torch_ops.cpp over libpma.so).

The reference binds its native kernels as a pybind module of libtorch functions
(src/prime_moment_attention/prime_cpp_kernel.cpp:119-124).  Here they are dispatcher operators,
callable without ctypes and traceable by torch.compile / torch.export, which see each call as one
opaque node whose output shapes come from the fake implementations registered below.

    torch.ops.pma.prefill(q, k, v, decay, state=None, eps=1.0, return_state=True) -> (y, [state])
    torch.ops.pma.decode_step(q, k, v, decay, state, eps=1.0) -> (y, [new state])
    torch.ops.pma.decode_step_(q, k, v, decay, state, eps=1.0) -> y        (state updated in place)

    torch.ops.pma.gated_scan, gated_scan_step, gated_scan_step_, sample, fp8_linear: the calls behind
    the recurrence, sampling and fp8 modules, which document their arguments

`decay` is a float32 CUDA tensor of H (or B*H) decays; states are the reference tuple
(S0, S1, S2, K0, K1, K2) in float32.  Loading fails loudly when _pma_torch.so is missing.
"""
from __future__ import annotations

import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "_pma_torch.so")
_loaded = False
_watching = False


def _state_like(B: int, H: int, D: int, device):
    f = lambda *s: torch.empty(*s, dtype=torch.float32, device=device)  # noqa: E731
    return [f(B, H, D), f(B, H, D, D), f(B, H, D, D), f(B, H, 1), f(B, H, D), f(B, H, D)]


def _scan_bytes(words: int) -> int:
    """pma_gated_scan_workspace_bytes of `words` states: 256 + states, then runs, each rounded to 256."""
    runs_at = (256 + 4 * words + 255) // 256 * 256
    return (runs_at + 8 * words + 255) // 256 * 256


# (run, not traced, where torch.compile meets it: a program's first use may be inside a compiled function)
@torch.compiler.assume_constant_result
def load() -> None:
    """Load the operator library (once) and register the operators' shape functions."""
    global _loaded
    if _loaded:
        return
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python -m prime_moment_attention_b200.build`")
    torch.ops.load_library(LIB_PATH)

    @torch.library.register_fake("pma::prefill")
    def _prefill_fake(q, k, v, decay, state=None, eps=1.0, return_state=True):
        B, H, L, D = q.shape
        return q.new_empty(B, H, L, D), (_state_like(B, H, D, q.device) if return_state else [])

    @torch.library.register_fake("pma::decode_step")
    def _decode_fake(q, k, v, decay, state, eps=1.0):
        N, H, D = q.shape
        return q.new_empty(N, H, D), _state_like(N, H, D, q.device)

    @torch.library.register_fake("pma::decode_step_")
    def _decode_inplace_fake(q, k, v, decay, state, eps=1.0):
        return q.new_empty(q.shape)

    @torch.library.register_fake("pma::gated_scan")
    def _gated_scan_fake(x, f, bias=None, gate=None, h0=None, reset=None):
        return x.new_empty(x.shape), x.new_empty((x.shape[0], x.shape[2]), dtype=torch.float32)

    @torch.library.register_fake("pma::gated_scan_forward")
    def _gated_scan_forward_fake(x, f, bias, gate, h0, reset):
        B, L, C = x.shape
        words = B * ((L + 127) // 128) * C
        return (x.new_empty(x.shape), x.new_empty((B, C), dtype=torch.float32),
                x.new_empty((0 if L <= 128 else _scan_bytes(words),), dtype=torch.uint8))

    @torch.library.register_fake("pma::gated_scan_backward")
    def _gated_scan_backward_fake(x, f, bias, gate, h0, reset, ws, dy, dh, want_bias, want_h0):
        B, _, C = x.shape
        f32 = lambda *s: x.new_empty(s, dtype=torch.float32)  # noqa: E731
        return (x.new_empty(x.shape), x.new_empty(x.shape), f32(C) if want_bias else f32(0),
                x.new_empty(x.shape if gate is not None else (0,)), f32(B, C) if want_h0 else f32(0))

    @torch.library.register_fake("pma::gated_scan_step")
    def _gated_scan_step_fake(x, f, h, bias=None, gate=None):
        return x.new_empty(x.shape), h.new_empty(h.shape)

    @torch.library.register_fake("pma::gated_scan_step_")
    def _gated_scan_step_inplace_fake(x, f, h, bias=None, gate=None, rows=None):
        return x.new_empty(x.shape)

    @torch.library.register_fake("pma::sample")
    def _sample_fake(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, t=1.0, k=0, p=1.0, m=0.0):
        return u.new_empty(u.shape, dtype=torch.int64), u.new_empty(u.shape)

    @torch.library.register_fake("pma::fp8_linear")
    def _fp8_linear_fake(x, wq, ws, out_dtype):
        return x.new_empty((*x.shape[:-1], wq.shape[0]), dtype=out_dtype)

    _loaded = True


@torch.compiler.assume_constant_result
def watch_faults() -> None:
    """Load, and let the operators whose kernels wait (the recurrence's tiles, the 8-bit product) look at the
    fault word themselves: a compiled program calls them without the Python layer's check."""
    global _watching
    if not _watching:
        from . import ops
        direct().watch_faults(ops.fault_address())
        _watching = True


def direct():
    """The extension module of the layer operators: the same functions, called without the dispatcher's
    boxing.  Its functions return NotImplemented for what the dispatcher has to see."""
    load()
    from . import _pma_torch
    return _pma_torch


def prefill(q, k, v, decay: torch.Tensor, state=None, eps: float = 1.0, return_state: bool = True):
    """torch.ops.pma.prefill with the library loaded; returns (y, state tuple or None)."""
    load()
    y, st = torch.ops.pma.prefill(q, k, v, decay, None if state is None else list(state), eps, return_state)
    return y, (tuple(st) if return_state else None)


def decode_step(q, k, v, decay: torch.Tensor, state, eps: float = 1.0, inplace: bool = False):
    """torch.ops.pma.decode_step (functional) or decode_step_ (inplace); returns (y, state tuple)."""
    load()
    if inplace:
        return torch.ops.pma.decode_step_(q, k, v, decay, list(state), eps), tuple(state)
    y, st = torch.ops.pma.decode_step(q, k, v, decay, list(state), eps)
    return y, tuple(st)
