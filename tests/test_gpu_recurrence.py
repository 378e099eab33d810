"""The gated recurrence kernels against the float64 statement of tests/recurrence_oracle.py.

Tolerances.  A relative error d in every z_t moves h by at most d times the range of x and h0 (h is
a convex combination of them).  d is below 2e-6 for |f + bias| <= 20: the float32 sum (half an ulp
of 20, 1e-6), the scaled exponent (half an ulp of 29 times ln 2, 7e-7) and 2^-22 each from the
exponential and the reciprocal.  The joins add an ulp of the state a tile, damped by the decay:
below 2e-6 of the range at the lengths here.  Four times their sum, 2e-5 of the range, is the
bar for h in float32; gradients carry two such factors (the states and the carries) and get 4e-5 of their largest
value.  bf16 outputs add one rounding, 2^-9 of the value itself.
"""
import numpy as np
import pytest
import torch

from prime_moment_attention_b200 import _lib, ops, recurrence
from tests.recurrence_oracle import recurrence as oracle

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _inputs(B, L, C, dtype, gate=True, bias=True, h0=True, reset=False, layout="own", seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 7 * L + C)
    dt = DT[dtype]
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    n = 2 + int(gate)
    if layout == "packed":      # column slices of one projection
        p = r(B, L, n * C).to(dt).cuda()
        parts = [p[..., i * C:(i + 1) * C] for i in range(n)]
    elif layout == "time":      # [L, B, C] storage
        parts = [r(L, B, C).to(dt).cuda().transpose(0, 1) for _ in range(n)]
    elif layout == "offset":    # rows that start on no vector boundary
        parts = [r(B, L, C + 3).to(dt).cuda()[..., 1:1 + C] for _ in range(n)]
    else:
        parts = [r(B, L, C).to(dt).cuda() for _ in range(n)]
    parts[1].mul_(spread)
    a = {"x": parts[0], "f": parts[1], "gate": parts[2] if gate else None,
         "bias": (torch.rand(C, generator=g) * 9.0).cuda() if bias else None,
         "h0": r(B, C).cuda() if h0 else None, "reset": None}
    if reset:
        a["reset"] = (torch.rand(B, L, generator=g) < 0.05).cuda()
    return a, r(B, L, C).to(dt).cuda(), r(B, C).cuda()


def _close(got, want, tol, name, dtype=torch.float32, scale=None):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, name
    scale = np.abs(want).max(initial=0.0) if scale is None else scale
    bar = tol * scale + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0.0) + 1e-30
    bad = np.abs(got - want) > bar
    assert not bad.any(), (name, int(bad.sum()), float(np.abs(got - want).max()), float(scale))


CASES = [
    (1, 1, 1, "f32", {}), (2, 3, 5, "bf16", {}), (1, 127, 64, "bf16", {}), (2, 128, 64, "bf16", {}),
    (1, 129, 66, "bf16", {"reset": True}), (3, 300, 33, "bf16", {"layout": "offset"}),
    (2, 1000, 96, "f32", {"reset": True, "layout": "packed"}), (1, 4099, 40, "f32", {"gate": False}),
    (2, 257, 128, "bf16", {"gate": False, "bias": False, "h0": False}), (4, 640, 70, "bf16", {"layout": "time"}),
    (1, 2500, 1, "bf16", {"layout": "packed"}), (2, 2176, 30, "f32", {"h0": False, "layout": "offset"}),
    (1, 20000, 64, "bf16", {"layout": "packed"}),
    # more tiles than fit the GPU at once, with and without the strides that TMA takes
    (2, 5000, 1024, "bf16", {"layout": "packed", "reset": True}), (1, 5000, 1024, "f32", {}),
    (2, 3000, 1001, "bf16", {}),
    # two to eight tiles, as a cluster and otherwise
    (1, 1024, 64, "bf16", {"reset": True}), (3, 385, 96, "f32", {"gate": False, "reset": True}),
    (16, 900, 256, "bf16", {"layout": "packed"}), (1, 1025, 64, "bf16", {}),
]


@pytest.mark.parametrize("B,L,C,dtype,opts", CASES)
def test_forward_and_gradients(B, L, C, dtype, opts):
    a, dy, dh = _inputs(B, L, C, dtype, **opts)
    want = oracle(a["x"], a["f"], a["bias"], a["gate"], a["h0"], a["reset"], dy, dh)
    names = [k for k in ("x", "f", "bias", "gate", "h0") if a[k] is not None]
    for k in names:
        a[k] = a[k].detach().requires_grad_()
    y, h = recurrence.gated_scan(a["x"], a["f"], a["bias"], a["gate"], a["h0"], a["reset"])
    grads = dict(zip(names, torch.autograd.grad([y, h], [a[k] for k in names], [dy, dh])))
    dt = DT[dtype]
    span = max(float(a["x"].abs().max()), float(a["h0"].abs().max()) if a["h0"] is not None else 0.0)
    _close(h, want["h"], 2e-5, "h", scale=span)
    _close(y, want["y"], 2e-5, "y", dt, scale=span * (1 if a["gate"] is None else max(1.0, float(a["gate"].abs().max()))))
    for k in names:
        if k == "bias":  # a sum: relative to the sum of magnitudes
            _close(grads[k], want["dbias"], 1.0, "dbias", scale=4e-5 * want["dbias_abs"])
        else:
            _close(grads[k], want["d" + k], 4e-5, "d" + k, torch.float32 if k == "h0" else dt)


def test_results_and_gradients_repeat_bit_for_bit():
    a, dy, dh = _inputs(2, 9000, 64, "bf16", reset=True)
    names = ("x", "f", "bias", "gate", "h0")
    for k in names:
        a[k] = a[k].detach().requires_grad_()
    first = None
    for _ in range(5):
        y, h = recurrence.gated_scan(*(a[k] for k in names), a["reset"])
        got = [y, h, *torch.autograd.grad([y, h], [a[k] for k in names], [dy, dh])]
        if first is None:
            first = got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_directional_derivative_of_the_kernel():
    """(L(p + e d) - L(p - e d)) / 2e against <grad, d> in float32.  The loss is a sum of 60 thousand
    terms near 1, computed to 2e-6 of the range each and added in float64: its noise is below
    sqrt(6e4) 4e-6 / 2e = 0.05 at e = 1e-2; the truncation e^2 L''' / 6 is of the same order.  The
    derivative along a random direction is some tens to hundreds: the bar is 0.5."""
    a, dy, dh = _inputs(2, 500, 60, "f32", reset=True)
    names = ("x", "f", "bias", "gate", "h0")
    for k in names:
        a[k] = a[k].detach().requires_grad_()

    def loss(shift, d):
        with torch.no_grad():
            y, h = recurrence.gated_scan(*(a[k] + shift * d[k] for k in names), a["reset"])
            return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    y, h = recurrence.gated_scan(*(a[k] for k in names), a["reset"])
    grads = torch.autograd.grad([y, h], [a[k] for k in names], [dy, dh])
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        d = {k: torch.randn(a[k].shape, generator=g).cuda() for k in names}
        want = sum(float((gr.double() * d[k].double()).sum()) for k, gr in zip(names, grads))
        num = (loss(1e-2, d) - loss(-1e-2, d)) / 2e-2
        assert abs(num - want) < 0.5, (num, want)


@pytest.mark.parametrize("dtype,C", [("bf16", 64), ("bf16", 33), ("f32", 40)])
def test_steps_continue_a_scan(dtype, C):
    a, _, _ = _inputs(3, 150, C, dtype, layout="packed")
    want = oracle(a["x"], a["f"], a["bias"], a["gate"], a["h0"])
    _, h = recurrence.gated_scan(a["x"][:, :140], a["f"][:, :140], a["bias"], a["gate"][:, :140], a["h0"])
    span = 6.0
    for t in range(140, 150):
        before = h.clone()
        y, h2 = recurrence.gated_scan_step(a["x"][:, t], a["f"][:, t], h, bias=a["bias"], gate=a["gate"][:, t])
        assert torch.equal(h, before)  # functional by default
        y2, h = recurrence.gated_scan_step(a["x"][:, t], a["f"][:, t], h, bias=a["bias"], gate=a["gate"][:, t],
                                           inplace=True)
        assert torch.equal(y, y2) and torch.equal(h, h2)
        _close(y, want["y"][:, t], 2e-5, "y", DT[dtype], scale=span * 4)
    _close(h, want["h"], 2e-5, "h", scale=span)


def test_step_over_pool_rows():
    a, _, _ = _inputs(4, 1, 64, "bf16")
    pool = torch.randn(6, 64).cuda()
    rows = torch.tensor([5, 0, -1, 9], dtype=torch.int32).cuda()  # two rows outside the pool
    x, f, gate = a["x"][:, 0], a["f"][:, 0], a["gate"][:, 0]
    before = pool.clone()
    y, got = recurrence.gated_scan_step(x, f, pool, bias=a["bias"], gate=gate, rows=rows)
    assert got.data_ptr() == pool.data_ptr()
    yw, hw = recurrence.gated_scan_step(x[:2], f[:2], before[[5, 0]], bias=a["bias"], gate=gate[:2])
    assert torch.equal(y[:2], yw) and torch.equal(pool[[5, 0]], hw)
    assert not y[2:].any() and torch.equal(pool[1:5], before[1:5])


def test_empty_and_split_sequences():
    a, _, _ = _inputs(2, 700, 48, "f32", reset=True)
    y, h = recurrence.gated_scan(a["x"][:, :0], a["f"][:, :0], h0=a["h0"])
    assert y.shape == (2, 0, 48) and torch.equal(h, a["h0"])
    assert not recurrence.gated_scan(a["x"][:, :0], a["f"][:, :0])[1].any()
    assert recurrence.gated_scan(a["x"][:0], a["f"][:0])[0].shape == (0, 700, 48)
    # two calls that hand the state over agree with one
    y, h = recurrence.gated_scan(a["x"], a["f"], a["bias"], a["gate"], a["h0"], a["reset"])
    cut = lambda t, s: None if t is None else t[:, s]  # noqa: E731
    s1, s2 = slice(0, 333), slice(333, 700)
    y1, h1 = recurrence.gated_scan(cut(a["x"], s1), cut(a["f"], s1), a["bias"], cut(a["gate"], s1), a["h0"],
                                   cut(a["reset"], s1))
    y2, h2 = recurrence.gated_scan(cut(a["x"], s2), cut(a["f"], s2), a["bias"], cut(a["gate"], s2), h1,
                                   cut(a["reset"], s2))
    torch.testing.assert_close(torch.cat([y1, y2], 1), y, rtol=0, atol=4e-5 * 6 * 4)
    torch.testing.assert_close(h2, h, rtol=0, atol=4e-5 * 6)


def test_extreme_gates_and_values():
    """Saturated gates: f = +-inf and +-1e4 give a = 1 or 0 exactly; a reset shields later tokens from
    a NaN or an infinite state before it, in both directions."""
    B, L, C = 1, 260, 8
    x = torch.randn(B, L, C).cuda()
    f = torch.zeros(B, L, C).cuda()
    f[:, :, 0], f[:, :, 1], f[:, :, 2], f[:, :, 3] = 1e4, -1e4, float("inf"), float("-inf")
    h0 = torch.randn(B, C).cuda()
    x.requires_grad_(), f.requires_grad_()
    y, h = recurrence.gated_scan(x, f, h0=h0)
    torch.testing.assert_close(y[0, :, 0], h0[0, 0].expand(L), rtol=0, atol=1e-30)
    torch.testing.assert_close(y[0, :, 2], h0[0, 2].expand(L), rtol=0, atol=1e-30)
    assert torch.equal(y[0, :, 1], x[0, :, 1]) and torch.equal(y[0, :, 3], x[0, :, 3])
    dx, df = torch.autograd.grad(y, [x, f], torch.ones_like(y))
    assert torch.isfinite(dx).all() and torch.isfinite(df).all()
    bad = x.detach().clone()
    bad[:, 50] = float("nan")
    bad[:, 51, :4] = float("inf")
    reset = torch.zeros(B, L, dtype=torch.uint8).cuda()
    reset[:, 200] = 1
    y, h = recurrence.gated_scan(bad, torch.randn(B, L, C).cuda(), h0=h0, reset=reset)
    assert torch.isfinite(y[:, 200:]).all() and torch.isfinite(h).all()


def test_runs_in_a_thread_without_a_context():
    """A thread whose first CUDA call is ours (an autograd worker is one)."""
    import threading
    a, _, _ = _inputs(1, 100, 64, "f32")
    want = recurrence.gated_scan(a["x"], a["f"], h0=a["h0"])
    got = []
    t = threading.Thread(target=lambda: got.extend(recurrence.gated_scan(a["x"], a["f"], h0=a["h0"])))
    t.start()
    t.join()
    assert len(got) == 2 and all(torch.equal(p, q) for p, q in zip(want, got))


def test_runs_on_the_current_stream():
    a, _, _ = _inputs(2, 600, 64, "bf16")
    want = recurrence.gated_scan(a["x"], a["f"], a["bias"], a["gate"], a["h0"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = recurrence.gated_scan(a["x"], a["f"], a["bias"], a["gate"], a["h0"])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_expired_wait_is_reported():
    """The test hook makes a launch give up before any work; the fault word carries the code."""
    a, _, _ = _inputs(1, 600, 64, "bf16")
    ops.check_faults(synchronize=True)
    _lib.load().pma_test_expire_waits(1_000_000)
    try:
        recurrence.gated_scan(a["x"], a["f"])
    finally:
        _lib.load().pma_test_expire_waits(0)
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelFault) as e:
        recurrence.gated_scan(a["x"], a["f"])
    assert e.value.code == 120
    recurrence.gated_scan(a["x"], a["f"])
    ops.check_faults(synchronize=True)


def test_offsets_past_32_bits():
    """More than 2^31 elements a tensor, forward and backward: the last tokens against a call on them
    alone that starts from the state before them (and, for the gradient, ends as the long one does)."""
    B, L, C = 1, 2200000, 1024
    cut = L - 1000 - (L - 1000) % 128
    x, f = (torch.empty(B, L, C, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(2))
    x.requires_grad_()
    bias = torch.full((C,), 3.0, device="cuda")
    y, h = recurrence.gated_scan(x, f, bias)
    dy = torch.ones(1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(B, L, C)
    (dx,) = torch.autograd.grad([y], [x], [dy])
    with torch.no_grad():
        _, before = recurrence.gated_scan(x[:, :cut], f[:, :cut], bias)
    tail = x[:, cut:].detach().requires_grad_()
    y2, h2 = recurrence.gated_scan(tail, f[:, cut:], bias, h0=before)
    (dx2,) = torch.autograd.grad([y2], [tail], [torch.ones_like(y2)])
    # states within the bar of the module's docstring (values are below 6), rounded to bf16
    torch.testing.assert_close(h2, h, rtol=0, atol=2e-4)
    torch.testing.assert_close(y2.float(), y[:, cut:].float(), rtol=2.0 ** -8, atol=2e-4)
    torch.testing.assert_close(dx2.float(), dx[:, cut:].float(), rtol=2.0 ** -8, atol=2e-4)


# float32 rows of a width that TMA takes, and of one that it does not; bf16 pairs and single channels
REPEATS = [(2, 9000, 64, "bf16"), (2, 9000, 66, "bf16"), (2, 9000, 33, "bf16"), (2, 9000, 64, "f32"), (2, 9000, 33, "f32"),
           (1, 40000, 256, "bf16"), (2, 900, 64, "bf16"), (2, 900, 33, "f32")]


@pytest.mark.parametrize("B,L,C,dtype", REPEATS)
@pytest.mark.parametrize("bias", [0.0, 2.2])
def test_results_repeat_without_resets(B, L, C, dtype, bias):
    """Whether a tile finds a neighbour's state or its run must not show: bit for bit the same, also where a tile forgets
    all that entered it, with a large state, and with a NaN early on."""
    a, dy, dh = _inputs(B, L, C, dtype, bias=False, spread=1.0)
    a["bias"] = torch.full((C,), bias).cuda()
    a["h0"] = a["h0"] * 1e6
    a["x"][0, 200, 0] = float("nan")
    dh = dh * 1e6
    names = ("x", "f", "bias", "gate", "h0")
    for k in names:
        a[k] = a[k].detach().requires_grad_()
    first = None
    for _ in range(12):
        y, h = recurrence.gated_scan(*(a[k] for k in names))
        got = [y, h, *torch.autograd.grad([y, h], [a[k] for k in names], [dy, dh])]
        bits = [t.detach().nan_to_num(nan=-12345.0) for t in got]
        first = first or bits
        assert all(torch.equal(p, q) for p, q in zip(first, bits))


# tiles by TMA, without it, and as a cluster; float32 states throughout
LARGE = [(1, 2560, 64, "f32"), (1, 2560, 33, "f32"), (1, 2560, 64, "bf16"), (1, 1000, 64, "f32"), (1, 1000, 33, "bf16")]


@pytest.mark.parametrize("reset", [False, True])
@pytest.mark.parametrize("B,L,C,dtype", LARGE)
def test_a_large_state_is_forgotten(B, L, C, dtype, reset):
    """h0 = 1e8 (and dh = 1e8 from the right) under a = 1/2 and x = 1: as in a token-by-token loop the error
    follows the state as it decays.  A row changes it by at most 2^-22 of its size (a within 2^-23, two
    roundings) and 1e8 is below 1 after 27 rows: 7e-6 of |h_t| + 1, a third of the bar of 2e-5."""
    x, f = torch.ones(B, L, C, dtype=DT[dtype]).cuda(), torch.zeros(B, L, C, dtype=DT[dtype]).cuda()
    h0, dh = torch.full((B, C), 1e8).cuda(), torch.full((B, C), 1e8).cuda()
    cut = None
    if reset:  # the variant with resets, none of them here
        cut = torch.zeros(B, L, dtype=torch.bool).cuda()
    dy = torch.ones_like(x)
    want = oracle(x, f, None, None, h0, cut, dy, dh)
    x.requires_grad_(), f.requires_grad_(), h0.requires_grad_()
    y, h = recurrence.gated_scan(x, f, h0=h0, reset=cut)
    dx, d0 = torch.autograd.grad([y, h], [x, h0], [dy, dh])
    half = 2.0 ** -8 if dtype == "bf16" else 0.0
    for got, w, r in ((y, want["y"], half), (h, want["h"], 0.0), (dx, want["dx"], half), (d0, want["dh0"], 0.0)):
        got = got.detach().double().cpu().numpy()
        assert (np.abs(got - w) <= (2e-5 + r) * (np.abs(w) + 1.0)).all()


@pytest.mark.parametrize("reset", [False, True])
@pytest.mark.parametrize("B,L,C,dtype", LARGE)
def test_a_nan_stays_until_a_reset(B, L, C, dtype, reset):
    """Decays of all sizes: a NaN at token 150 reaches every later token of its channel, up to a reset at
    token 700 where there is one, and no earlier token and no other channel."""
    a, _, _ = _inputs(B, L, C, dtype, gate=False, bias=False, spread=3.0)
    a["x"][0, 150, 3] = float("nan")
    cut = None
    if reset:
        cut = torch.zeros(B, L, dtype=torch.bool).cuda()
        cut[0, 700] = True
    y, h = recurrence.gated_scan(a["x"], a["f"], h0=a["h0"], reset=cut)
    nan = torch.zeros(L, C, dtype=torch.bool)
    nan[150:700 if reset else L, 3] = True
    assert torch.equal(torch.isnan(y[0]).cpu(), nan)
    assert torch.equal(torch.isnan(h[0]).cpu(), nan[-1])
