"""Argument checks of the 8-bit product: nothing here touches a device."""
import pytest
import torch

from prime_moment_attention_b200 import _lib, fp8


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4)
    q = x.to(torch.float8_e4m3fn)
    for call in (lambda: fp8.quantize(x), lambda: fp8.quantize_weight(x), lambda: fp8.linear(x, q, x[:1, :1]),
                 lambda: fp8.matmul(q, x[:, :1], q, x[:1, :1])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("change,status", [
    (dict(M=-1), 1), (dict(N=0), 1), (dict(K=0), 1), (dict(xq=None), 1), (dict(xq=260), 4), (dict(xq_stride=260), 4),
    (dict(wq_stride=240), 4), (dict(xs=None), 1), (dict(ws_stride=1), 1), (dict(y=None), 1), (dict(y_stride=63), 1),
    (dict(dt=5), 3), (dict(y=257), 4),
])
def test_matmul_argument_errors(change, status):
    a = dict(M=4, N=64, K=256, xq=256, xq_stride=256, xs=256, wq=256, wq_stride=256, ws=256, ws_stride=2, y=256,
             y_stride=64, dt=_lib.PMA_BF16)
    a.update(change)
    rc = _lib.load().pma_fp8_matmul(a["M"], a["N"], a["K"], a["xq"], a["xq_stride"], a["xs"], 1, a["M"], a["wq"],
                                    a["wq_stride"], a["ws"], a["ws_stride"], a["y"], a["y_stride"], a["dt"], None)
    assert rc == status


def test_linear_needs_its_workspace():
    L = _lib.load()
    n = L.pma_fp8_linear_workspace_bytes(3, 200)
    assert n >= 3 * 208 + 3 * 2 * 4
    for ws, size in ((None, n), (256, n - 1), (264, n)):
        assert L.pma_fp8_linear(3, 64, 200, 256, 200, _lib.PMA_BF16, 256, 208, 256, 2, 256, 64, _lib.PMA_BF16, ws, size,
                                None) == 5
