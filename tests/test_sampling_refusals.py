"""Argument checks of the sampler: nothing here touches a device."""
import pytest
import torch

from prime_moment_attention_b200 import _lib, sampling


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        sampling.sample(torch.zeros(1, 4), torch.zeros(1))


@pytest.mark.parametrize("change,status", [
    (dict(B=-1), 1), (dict(V=0), 1), (dict(V=360449), 1), (dict(stride=10), 1), (dict(dtype=7), 3),
    (dict(logits=None), 1), (dict(u=None), 1), (dict(tokens=None), 1), (dict(logits=257), 4),
])
def test_argument_errors(change, status):
    a = dict(B=2, V=100, logits=256, stride=100, dtype=_lib.PMA_F32, u=256, tokens=256)
    a.update(change)
    rc = _lib.load().pma_sample(a["B"], a["V"], a["logits"], a["stride"], a["dtype"], a["u"], None, 1.0, None, 0, None,
                                1.0, None, 0.0, a["tokens"], None, None)
    assert rc == status
