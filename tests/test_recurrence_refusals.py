"""Argument checks of the gated recurrence: nothing here touches a device."""
import ctypes

import pytest
import torch

from prime_moment_attention_b200 import _lib, recurrence


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        recurrence.gated_scan(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        recurrence.gated_scan_step(x[0], x[0], torch.zeros(2, 3))


def _t(dt=_lib.PMA_BF16, ptr=256, sb=64, sl=64):
    return ctypes.byref(_lib.SeqTensor(ptr, dt, sb, 0, sl))


@pytest.mark.parametrize("change,status", [
    ({"B": -1}, 1), ({"C": 0}, 1), ({"x": None}, 1), ({"f": _t(_lib.PMA_F32)}, 3), ({"x": _t(9)}, 3),
    ({"y": _t(ptr=0)}, 1), ({"gate": _t(ptr=257)}, 4), ({"f": _t(sl=-64)}, 4),
])
def test_forward_argument_errors(change, status):
    a = {"B": 1, "L": 300, "C": 64, "x": _t(), "f": _t(), "gate": None, "y": _t(), **change}
    rc = _lib.load().pma_gated_scan(a["B"], a["L"], a["C"], a["x"], a["f"], a["gate"], None, None, None, a["y"], None,
                                    None, 0, None)
    assert rc == status


def test_backward_gate_and_its_gradient_go_together():
    rc = _lib.load().pma_gated_scan_backward(1, 300, 64, _t(), _t(), _t(), None, None, None, _t(), None, _t(), _t(),
                                             None, None, None, None, 0, None, 0, None)
    assert rc == 1


def test_workspace_sizes():
    L = _lib.load()
    assert L.pma_gated_scan_workspace_bytes(4, 128, 64) == 0  # one tile: nothing to hand over
    assert L.pma_gated_scan_workspace_bytes(4, 129, 64) >= 4 * 2 * 64 * 12
    # 64-bit sizes: 2^20 tokens of 4096 channels in 16 rows
    assert L.pma_gated_scan_workspace_bytes(16, 1 << 20, 4096) > 6 << 30


def test_traced_workspace_sizes_are_the_librarys():
    """The shape function restates the library's rule, in whole numbers that may be symbols."""
    from prime_moment_attention_b200 import torch_ops
    L = _lib.load()
    for B in (1, 3, 16):
        for n in (1, 127, 128, 129, 300, 4096, 99999):
            for C in (1, 5, 64, 515, 4096):
                words = B * ((n + 127) // 128) * C
                assert (0 if n <= 128 else torch_ops._scan_bytes(words)) == L.pma_gated_scan_workspace_bytes(B, n, C)


def test_states_in_place_are_refused():
    """The last state's tile may finish before every warp of the first has read the first state."""
    L = _lib.load()
    assert L.pma_gated_scan(1, 300, 64, _t(), _t(), None, None, 512, None, _t(), 512, 256, 1 << 20, None) == 1
    for dh_last, h0 in ((512, None), (None, 512)):
        assert L.pma_gated_scan_backward(1, 300, 64, _t(), _t(), None, None, h0, None, _t(), dh_last, _t(), _t(), None,
                                         None, 512, 256, 1 << 20, 256, 1 << 20, None) == 1
