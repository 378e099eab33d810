"""8-bit linear products for serving: e4m3 with a float32 scale per block of 128 (pma_fp8_*).

    wq, ws = quantize_weight(linear.weight)      # once: [N, K] e4m3, [ceil(N/128), ceil(K/128)]
    y = fp8.linear(x, wq, ws)                    # x [..., K] is quantised inside the call

Weights take half the bytes of bf16, and the tensor cores run e4m3 at twice the rate of bf16: products of
many tokens are faster than in bf16 (777 x 1530 x 1000 12 against 26 us, 8192^3 565 against 690); those of a
decode step save memory only (64 x 32000 x 768 12 against 7 us).  Inference only.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib, torch_ops
from .ops import _DT, _require_cuda, _stream, check_faults

E4M3 = torch.float8_e4m3fn
BLOCK = 128
_c = None


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _storage(rows: int, K: int, dev) -> torch.Tensor:
    """[rows, K] e4m3 whose rows start on 16-byte boundaries."""
    return torch.empty(rows, -(-K // 16) * 16, dtype=E4M3, device=dev)[:, :K]


def _inference_only(name: str, *ts: torch.Tensor) -> None:
    """No gradient or tangent is dropped in silence."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError(f"{name} is inference-only: run under torch.no_grad() or torch.inference_mode()")
    if any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{name} has no forward-mode derivative")


def _dense(name: str, x: torch.Tensor) -> torch.Tensor:
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"{name} must be a matrix with at least one column; got {tuple(x.shape)}")
    if x.dtype not in _DT:
        raise TypeError(f"unsupported dtype {x.dtype}: float32 or bfloat16")
    x = x.detach()
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _rows(name: str, q: torch.Tensor, K: int) -> torch.Tensor:
    if q.dim() != 2 or q.dtype != E4M3 or q.shape[1] != K:
        raise ValueError(f"{name} must be a [rows, {K}] float8_e4m3fn tensor")
    if q.stride(1) != 1 or q.stride(0) % 16 or q.stride(0) < K or q.data_ptr() % 16:
        aligned = _storage(q.shape[0], K, q.device)
        aligned.copy_(q)
        return aligned
    return q


def _scales(name: str, s: torch.Tensor, shape, dev) -> torch.Tensor:
    if tuple(s.shape) != tuple(shape) or s.dtype != torch.float32 or s.device != dev:
        raise ValueError(f"{name} must be a float32 tensor of shape {tuple(shape)} on {dev}")
    return s


class Fp8Weight:
    """A weight [N, K] kept in e4m3 with its block scales: call it on x [..., K]."""

    def __init__(self, weight: torch.Tensor):
        self.q, self.scale = quantize_weight(weight)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return linear(x, self.q, self.scale, out_dtype=x.dtype)


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[M, K] bf16 or float32 -> (e4m3 [M, K], scales [M, ceil(K/128)]).  The scales' storage is
    [ceil(K/128), M], the order the product reads them in.  Elements are e4m3(448 x / amax) of float32
    arithmetic, with amax the largest magnitude of a row's 128."""
    dev = _require_cuda(x)
    _inference_only("fp8.quantize", x)
    x = _dense("x", x)
    M, K = x.shape
    q, s = _storage(M, K, dev), torch.empty(_blocks(K), M, dtype=torch.float32, device=dev).t()
    _lib.check("pma_fp8_quantize", _lib.load().pma_fp8_quantize(
        M, K, x.data_ptr(), x.stride(0), _DT[x.dtype], q.data_ptr(), q.stride(0), s.data_ptr(), 1, M, _stream(dev)))
    return q, s


def quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[N, K] bf16 or float32 -> (e4m3 [N, K], scales [ceil(N/128), ceil(K/128)]).  A parameter is taken
    as it is, without its gradient."""
    dev = _require_cuda(w)
    w = _dense("w", w)
    N, K = w.shape
    q, s = _storage(N, K, dev), torch.empty(_blocks(N), _blocks(K), dtype=torch.float32, device=dev)
    _lib.check("pma_fp8_quantize_weight", _lib.load().pma_fp8_quantize_weight(
        N, K, w.data_ptr(), w.stride(0), _DT[w.dtype], q.data_ptr(), q.stride(0), s.data_ptr(), _stream(dev)))
    return q, s


def _out(out: Optional[torch.Tensor], M: int, N: int, dtype: torch.dtype, dev) -> torch.Tensor:
    if out is None:
        if dtype not in _DT:
            raise TypeError(f"unsupported dtype {dtype}: float32 or bfloat16")
        return torch.empty(M, N, dtype=dtype, device=dev)
    if (tuple(out.shape) != (M, N) or out.dtype not in _DT or out.device != dev or out.stride(1) != 1
            or (M > 1 and out.stride(0) < N)):
        raise ValueError(f"out must be a bf16 or float32 [{M}, {N}] tensor on {dev} with contiguous rows")
    return out


def matmul(xq: torch.Tensor, xs: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor,
           out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x @ w.T of quantised x [M, K] (scales [M, ceil(K/128)]) and w [N, K] (scales per 128 x 128)."""
    dev = _require_cuda(xq, xs, wq, ws)
    _inference_only("fp8.matmul", xs, ws)
    check_faults("fp8.matmul")
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] == 0:
        raise ValueError("xq and wq must be matrices with at least one column")
    (M, K), N = xq.shape, wq.shape[0]
    xq, wq = _rows("xq", xq, K), _rows("wq", wq, K)
    xs = _scales("xs", xs, (M, _blocks(K)), dev)
    ws = _scales("ws", ws, (_blocks(N), _blocks(K)), dev)
    # the kernel takes a row stride of at least K's blocks: a broadcast or overlapping view becomes an array of its own
    nb, kb = ws.shape
    if not ((kb == 1 or ws.stride(1) == 1) and (nb <= 1 or ws.stride(0) >= kb)):
        ws = ws.contiguous()
    y = _out(out, M, N, out_dtype, dev)
    if N and M:
        _lib.check("pma_fp8_matmul", _lib.load().pma_fp8_matmul(
            M, N, K, xq.data_ptr(), xq.stride(0), xs.data_ptr(), xs.stride(0), xs.stride(1), wq.data_ptr(),
            wq.stride(0), ws.data_ptr(), kb if nb <= 1 else ws.stride(0), y.data_ptr(), y.stride(0), _DT[y.dtype],
            _stream(dev)))
    return y


def linear(x: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] (bf16 or float32, quantised per row and 128 of K inside the call) times w [N, K] -> [..., N]."""
    global _c
    if out is None:
        if not torch.compiler.is_compiling() and out_dtype in _DT:
            if getattr(x, "is_cuda", False):
                check_faults("fp8.linear")
            if _c is None:
                _c = torch_ops.direct()
            r = _c.fp8_linear(x, wq, ws, out_dtype == torch.float32)
            if r is not NotImplemented:
                return r
        _require_cuda(x, wq, ws)
        torch_ops.watch_faults()
        return torch.ops.pma.fp8_linear.default(x, wq, ws, out_dtype)
    _require_cuda(x, wq, ws)
    if x.dim() != 2:
        raise ValueError("x must be a matrix when out is given")
    return matmul(*quantize(x), wq, ws, out=out)
