"""Token sampling on the GPU: temperature, top-k, top-p and min-p in one kernel (pma_sample).

The random numbers are given, one uniform float per row, so that a caller owns the generator, a
sampled step can be captured in a CUDA graph, and the same row with the same number gives the same
token in any batch.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from .ops import _DT, _require_cuda, _stream

Setting = Union[int, float, torch.Tensor]
MAX_VOCAB = 360448


def _setting(name: str, v: Setting, dtype: torch.dtype, B: int, dev) -> Tuple[Optional[torch.Tensor], Union[int, float]]:
    """(per-row tensor, 0) or (None, value for all rows)."""
    if isinstance(v, torch.Tensor):
        if v.shape != (B,) or v.device != dev or v.dtype != dtype:
            raise ValueError(f"{name} must be a number or a {dtype} tensor of shape ({B},) on {dev}")
        return v.contiguous(), 0
    return None, int(v) if dtype == torch.int32 else float(v)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
           top_p: Setting = 1.0, min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token per row of logits [B, V] (bf16 or float32); returns (tokens int64 [B], logprobs float32 [B]).

    u is float32 [B], uniform in [0, 1).  Settings are numbers or, one per row, tensors on the GPU
    (float32; int32 for top_k).  Tokens are ordered by (logit descending, index ascending) and cut
    by top_k, then by the smallest prefix that holds top_p of what is left, then by probability
    min_p times the largest; temperature 0 takes the most likely token.  The logprob is that of the
    token under softmax(logits / temperature) before any cut.  -inf and NaN logits are never taken;
    a row of nothing else gives token -1 and logprob -inf."""
    dev = _require_cuda(logits, u)
    if logits.dim() != 2 or logits.shape[1] == 0 or logits.shape[1] > MAX_VOCAB:
        raise ValueError(f"logits must be [B, V] with 1 <= V <= {MAX_VOCAB}; got {tuple(logits.shape)}")
    if logits.dtype not in _DT:
        raise TypeError(f"unsupported dtype {logits.dtype}: float32 or bfloat16")
    B, V = logits.shape
    if u.shape != (B,) or u.dtype != torch.float32:
        raise ValueError(f"u must be a float32 tensor of shape ({B},)")
    if logits.stride(1) != 1 and V > 1 or B > 1 and logits.stride(0) < V:
        logits = logits.contiguous()
    u = u.contiguous()
    (tt, tv), (kt, kv) = _setting("temperature", temperature, torch.float32, B, dev), _setting("top_k", top_k, torch.int32, B, dev)
    (pt, pv), (mt, mv) = _setting("top_p", top_p, torch.float32, B, dev), _setting("min_p", min_p, torch.float32, B, dev)
    tokens = torch.empty(B, dtype=torch.int64, device=dev)
    logprobs = torch.empty(B, dtype=torch.float32, device=dev)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check("pma_sample", _lib.load().pma_sample(
        B, V, logits.data_ptr(), logits.stride(0), _DT[logits.dtype], u.data_ptr(), ptr(tt), tv, ptr(kt), kv, ptr(pt),
        pv, ptr(mt), mv, tokens.data_ptr(), logprobs.data_ptr(), _stream(dev)))
    return tokens, logprobs
