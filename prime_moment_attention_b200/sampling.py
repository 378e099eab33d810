"""Token sampling on the GPU: temperature, top-k, top-p and min-p in one kernel (pma_sample).

The random numbers are given, one uniform float per row, so that a caller owns the generator, a
sampled step can be captured in a CUDA graph, and the same row with the same number gives the same
token in any batch.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Tuple, Union

import torch

from . import torch_ops
from .ops import _require_cuda

Setting = Union[int, float, torch.Tensor]
MAX_VOCAB = 360448
_c = None


@dataclass
class Sampler:
    """Settings of sample(), as numbers or per-row tensors."""
    temperature: Setting = 1.0
    top_k: Setting = 0
    top_p: Setting = 1.0
    min_p: Setting = 0.0

    def __call__(self, logits: torch.Tensor, u: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        return sample(logits, u, self.temperature, self.top_k, self.top_p, self.min_p)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
           top_p: Setting = 1.0, min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token per row of logits [B, V] (bf16 or float32); returns (tokens int64 [B], logprobs float32 [B]).

    u is float32 [B], uniform in [0, 1).  Settings are numbers or, one per row, tensors on the GPU
    (float32; int32 for top_k).  Tokens are ordered by (logit descending, index ascending) and cut
    by top_k, then by the smallest prefix that holds top_p of what is left, then by probability
    min_p times the largest; temperature 0 takes the most likely token.  The logprob is that of the
    token under softmax(logits / temperature) before any cut; it carries no gradient.  -inf and NaN logits are never taken;
    a row of nothing else gives token -1 and logprob -inf."""
    global _c
    if not torch.compiler.is_compiling():
        if _c is None:
            _c = torch_ops.direct()
        r = _c.sample(logits, u, temperature, top_k, top_p, min_p)
        if r is not NotImplemented:
            return r
    torch_ops.load()
    _require_cuda(logits, u)
    rows = [v if isinstance(v, torch.Tensor) else None for v in (temperature, top_k, top_p, min_p)]
    t, k, p, m = (v if r is None else 0 for v, r in zip((temperature, top_k, top_p, min_p), rows))
    return torch.ops.pma.sample.default(logits, u, *rows, t, k, p, m)
