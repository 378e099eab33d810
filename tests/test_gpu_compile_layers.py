"""The layer operators' Python functions inside torch.compile: whole graphs, in a process whose first use
of them is the compiled one, and their results those of the calls."""
import os
import subprocess
import sys

import pytest
import torch

from prime_moment_attention_b200 import _lib, fp8, ops, recurrence, sampling

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def scan(x, b, u, wq, ws):
    y, h = recurrence.gated_scan(x, x * 2, b, gate=x + 1)
    return (y * 2).sum() + h.sum()


def steps(x, b, u, wq, ws):
    y, h = recurrence.gated_scan_step(x[:, 0], x[:, 1], x[:, 2].clone(), bias=b)
    z, h2 = recurrence.gated_scan_step(x[:, 1], x[:, 2], h.clone(), bias=b, gate=x[:, 0], inplace=True)
    return y + z, h, h2


def tokens(x, b, u, wq, ws):
    t, p = sampling.sample(x[:, 0], u, temperature=0.8, top_k=20, top_p=0.9)
    t2, p2 = sampling.Sampler(temperature=b[:2], min_p=0.01)(x[:, 1], u)
    return t + t2, p + p2


def linear(x, b, u, wq, ws):
    return fp8.linear(x.bfloat16(), wq, ws) + 1, fp8.linear(x, wq, ws, out_dtype=torch.float32)


CALLS = {f.__name__: f for f in (scan, steps, tokens, linear)}


def _args(L=300):
    g = torch.Generator().manual_seed(L)
    x, b, u = torch.randn(2, L, 64, generator=g), torch.rand(64, generator=g), torch.rand(2, generator=g)
    w = (torch.randn(48, 64, generator=g) * 8).to(torch.float8_e4m3fn)
    return tuple(t.cuda() for t in (x, b, u, w, torch.ones(1, 1)))


def _same(p, q):
    p, q = ((v,) if isinstance(v, torch.Tensor) else v for v in (p, q))
    return all(torch.equal(a, b) for a, b in zip(p, q))


@pytest.mark.parametrize("name", sorted(CALLS))
def test_compiled_calls(name):
    with torch.no_grad():
        f = torch.compile(CALLS[name], backend="aot_eager", fullgraph=True)
        for L in (300, 50, 700):  # the length a symbol from the second on
            assert _same(f(*_args(L)), CALLS[name](*_args(L)))


def test_compiled_gradient():
    a = _args()
    got, want = [], []
    for f, out in ((torch.compile(scan, backend="aot_eager", fullgraph=True), got), (scan, want)):
        x, b = a[0].clone().requires_grad_(), a[1].clone().requires_grad_()
        out += torch.autograd.grad(f(x, b, *a[2:]), [x, b])
    assert _same(got, want)


@pytest.mark.parametrize("name", sorted(CALLS))
def test_the_first_use_may_be_compiled(name):
    code = (f"import torch, tests.test_gpu_compile_layers as t\nf = t.CALLS[{name!r}]\nwith torch.no_grad():\n"
            "    got = torch.compile(f, backend='aot_eager', fullgraph=True)(*t._args())\n"
            "    assert t._same(got, f(*t._args()))\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1500:]


@pytest.mark.parametrize("name,code", [("scan", 120), ("linear", 130)])
def test_a_compiled_program_sees_an_expired_wait(name, code):
    """The test hook makes a launch give up; the compiled program's next call says so, once."""
    with torch.no_grad():
        f = torch.compile(CALLS[name], backend="aot_eager", fullgraph=True)
        want = f(*_args())
        ops.check_faults(synchronize=True)
        _lib.load().pma_test_expire_waits(1_000_000)
        try:
            f(*_args())
        except RuntimeError:  # its own second launch may have seen the first's already
            pass
        finally:
            _lib.load().pma_test_expire_waits(0)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=f"fault code {code}"):
            f(*_args())
        assert _same(f(*_args()), want)
        ops.check_faults(synchronize=True)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", sorted(CALLS))
def test_traced_calls_are_calls(name):
    """torch.jit.trace records the operators, not their results on the example."""
    with torch.no_grad():
        f = torch.jit.trace(lambda *a: CALLS[name](*a), _args(), check_trace=False)
        other = tuple(a.flip(0) if i < 3 else a for i, a in enumerate(_args()))
        assert _same(f(*other), CALLS[name](*other)) and not _same(f(*other), f(*_args()))


@pytest.mark.filterwarnings("ignore")
def test_calls_under_vmap():
    x, b, u, wq, ws = _args()
    xs = torch.stack([x, x.flip(1), -x])
    with torch.no_grad():
        got = torch.func.vmap(lambda q: recurrence.gated_scan(q, q * 2, b))(xs)
        want = [recurrence.gated_scan(q, q * 2, b) for q in xs]
        assert all(torch.equal(got[i], torch.stack([w[i] for w in want])) for i in range(2))
