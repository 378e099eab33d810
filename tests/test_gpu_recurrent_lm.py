"""The recurrent model end to end: training gradients, prefill and steps, sampled decode in a graph on
8-bit weights, generate from given numbers."""
import pytest
import torch

from prime_moment_attention_b200 import fp8, recurrence, sampling
from prime_moment_attention_b200.model import DecodeGraph, PrimeConfig, PrimeForCausalLM

pytestmark = pytest.mark.gpu


def _model(dtype=torch.float32, vocab=301, seed=0):
    torch.manual_seed(seed)
    cfg = PrimeConfig(vocab_size=vocab, hidden_size=128, num_layers=2, num_heads=2, head_dim=64, use_recurrence=True,
                      initializer_range=0.1)
    return PrimeForCausalLM(cfg).cuda().to(dtype)


def _plain_scan(x, f, bias=None, gate=None, h0=None, reset=None):
    a = torch.sigmoid(f + bias)
    h = torch.zeros_like(x[:, 0]) if h0 is None else h0
    rows = []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        rows.append(h)
    return torch.stack(rows, 1) * torch.nn.functional.silu(gate), h


def test_training_gradients_match_a_plain_recurrence(monkeypatch):
    """float32 model, every parameter's gradient: the same network with the scan written in torch.  Both
    run the same float32 products elsewhere; the scan's own error is some 1e-6 of its range, amplified
    by two layers: 1e-4 of a gradient's largest value bounds it."""
    ids = torch.randint(301, (2, 150), device="cuda")
    grads = []
    for plain in (False, True):
        m = _model()
        if plain:
            monkeypatch.setattr(recurrence, "gated_scan", _plain_scan)
        m(ids, labels=ids)["loss"].backward()
        grads.append({n: p.grad for n, p in m.named_parameters()})
    assert all(g is not None for g in grads[0].values())
    for n, g in grads[0].items():
        want = grads[1][n]
        assert (g - want).abs().max() <= 1e-4 * want.abs().max() + 1e-9, n


def test_steps_and_prefill_agree():
    m = _model().eval()
    ids = torch.randint(301, (3, 40), device="cuda")
    with torch.no_grad():
        whole = m(ids)["logits"]
        out = m(ids[:, :33], return_states=True)
        states = out["states"]
        assert states[0][0].shape == (3, 128) and states[0][0].dtype == torch.float32
        for t in range(33, 40):
            out = m(ids[:, t:t + 1], states=states, return_states=True)
            states = out["states"]
            torch.testing.assert_close(out["logits"][:, 0], whole[:, t], rtol=1e-4, atol=1e-4)


def test_reset_separates_packed_documents():
    torch.manual_seed(3)
    layer = recurrence.GatedRecurrence(64).cuda()
    x = torch.randn(1, 50, 64, device="cuda")
    reset = torch.zeros(1, 50, dtype=torch.bool, device="cuda")
    reset[0, 20] = True
    with torch.no_grad():
        whole = layer(x, reset=reset)[0]
        torch.testing.assert_close(whole[:, 20:], layer(x[:, 20:])[0], rtol=1e-5, atol=1e-5)


class _PlainFp8Weight:
    """fp8.Fp8Weight written in torch: the same quantised values, the product in float32."""

    def __init__(self, weight):
        N, K = weight.shape
        q, s = fp8.quantize_weight(weight)
        self.w = q.float() * s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]

    def __call__(self, x):
        q, s = fp8.quantize(x)
        xd = q.float() * s.repeat_interleave(128, 1)[:, : x.shape[1]]
        return (xd @ self.w.t()).to(x.dtype)


@pytest.mark.parametrize("use_fp8", [False, True])
def test_sampled_decode_graph(use_fp8, monkeypatch):
    """The graph's logits against the eager model (bf16 products), or against a graph whose products are
    written in torch on the same quantised weights: what differs is bf16 rounding, 2^-9 an operation
    over some 20 of them in sequence and its effect on a few quantised elements: 2e-2 of the norm."""
    m = _model(torch.bfloat16).eval()
    ids = torch.randint(301, (5, 17), device="cuda")
    settings = sampling.Sampler(temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    with torch.no_grad():
        out = m(ids, return_states=True, last_logits_only=True)
        first = out["logits"][:, -1].argmax(-1)
        graph = DecodeGraph(m, out["states"], first, sampler=settings, fp8=use_fp8)
        if use_fp8:
            monkeypatch.setattr(fp8, "Fp8Weight", _PlainFp8Weight)
            plain = DecodeGraph(m, out["states"], first, sampler=settings, fp8=True)
        states, tok = out["states"], first
        for _ in range(6):
            u = torch.rand(5, generator=g, device="cuda")
            got = graph.step(u)[:, 0]
            if use_fp8:
                plain.tokens.copy_(tok[:, None])
                plain.step(u)
                want_logits = plain.logits
            else:
                eager = m(tok[:, None], states=states, return_states=True)
                states, want_logits = eager["states"], eager["logits"][:, 0]
            # the graph's token is what its own logits and u give
            want, lp = settings(graph.logits, u)
            assert torch.equal(got, want) and torch.equal(graph.logprobs, lp)
            err = (graph.logits.float() - want_logits.float()).norm() / want_logits.float().norm()
            assert err < 0.02, err
            tok = got.clone()
        with pytest.raises(ValueError, match="uniform"):
            graph.step()


def test_generate_from_given_numbers():
    m = _model().eval()
    ids = torch.randint(301, (4, 9), device="cuda")
    u = torch.rand(12, 4, device="cuda")
    a = m.generate(ids, max_new_tokens=12, temperature=0.9, top_k=30, top_p=0.95, uniforms=u)
    b = m.generate(ids, max_new_tokens=12, temperature=0.9, top_k=30, top_p=0.95, uniforms=u)
    assert a.shape == (4, 21) and torch.equal(a, b)
    alone = m.generate(ids[2:3], max_new_tokens=12, temperature=0.9, top_k=30, top_p=0.95, uniforms=u[:, 2:3])
    assert torch.equal(alone[0], a[2])
    assert torch.equal(m.generate(ids, max_new_tokens=3, temperature=0.0, uniforms=u),
                       m.generate(ids, max_new_tokens=3, temperature=0.0))
    with pytest.raises(ValueError, match="uniforms"):
        m.generate(ids, top_p=0.5)


@pytest.mark.parametrize("L", [50, 300])
def test_compile_sees_the_operators(L):
    """torch.compile traces the calls, and their gradient, as operators through their shape functions."""
    x = torch.randn(2, L, 64, device="cuda", requires_grad=True)
    b = torch.rand(64, device="cuda", requires_grad=True)
    scan = recurrence._ops()[0]

    def f(x, b):
        y, h = scan(x, x * 2, b, None, None, None)
        return (y * 2).sum() + h.sum()

    want = f(x, b)
    grads = torch.autograd.grad(want, [x, b])
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(x, b)
    assert torch.equal(want, got)
    for p, q in zip(grads, torch.autograd.grad(got, [x, b])):
        assert torch.equal(p, q)
    with torch.no_grad():
        assert torch.equal(want, torch.compile(f, backend="aot_eager", fullgraph=True)(x, b))


def test_calls_without_a_gradient_refuse_to_drop_it():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    h = torch.zeros(4, 64, device="cuda")
    q, s = fp8.quantize_weight(torch.randn(32, 64, device="cuda"))
    for call in (lambda: fp8.linear(x, q, s), lambda: recurrence.gated_scan_step(x, x, h),
                 lambda: recurrence.gated_scan_step(x, x, h, inplace=True)):
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
        with torch.no_grad():
            call()


def test_second_derivatives_are_refused():
    x = torch.randn(1, 10, 8, device="cuda", requires_grad=True)
    y, _ = recurrence.gated_scan(x, x)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad((y ** 2).sum(), x, create_graph=True)


@pytest.mark.parametrize("of", ["sum of y", "sum of h", "both", "square of y"])
def test_second_derivatives_are_refused_whatever_the_first_depends_on(of):
    """The gradient that enters may be a constant or belong to the last state alone: the gradients that
    leave depend on the inputs all the same, and carry no graph."""
    x = torch.randn(1, 300, 8, device="cuda", requires_grad=True)
    y, h = recurrence.gated_scan(x, x)
    loss = {"sum of y": y.sum(), "sum of h": (h ** 2).sum(), "both": y.sum() + h.sum(), "square of y": (y ** 2).sum()}[of]
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(loss, x, create_graph=True, retain_graph=True)
    assert torch.isfinite(torch.autograd.grad(loss, x)[0]).all()


def test_forward_mode_is_refused():
    """No tangent is dropped: a dual operand raises, in the direct call and through the dispatcher."""
    import torch.autograd.forward_ad as fwd
    x, f, gate = (torch.randn(2, 20, 8, device="cuda") for _ in range(3))
    bias, h0 = torch.randn(8, device="cuda"), torch.randn(2, 8, device="cuda")
    scan = recurrence._ops()[0]
    with fwd.dual_level():
        for i in range(5):
            ops = [x, f, bias, gate, h0]
            ops[i] = fwd.make_dual(ops[i], torch.ones_like(ops[i]))
            for call in (lambda: recurrence.gated_scan(*ops), lambda: scan(*ops, None)):
                for grad in (False, True):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                        call()
        ops = [x[:, 0], f[:, 0], h0, bias, gate[:, 0]]
        for i in range(5):
            dual = list(ops)
            dual[i] = fwd.make_dual(ops[i].contiguous(), torch.ones_like(ops[i]))
            for kw in ({}, {"inplace": True}):
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                    recurrence.gated_scan_step(*dual, **kw)
        q, s = fp8.quantize_weight(torch.randn(32, 8, device="cuda"))
        a = fwd.make_dual(x[0].clone(), torch.ones_like(x[0]))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
            fp8.linear(a, q, s)
    recurrence.gated_scan(x, f, bias, gate, h0)


@pytest.mark.parametrize("which", ["x", "f", "h", "bias", "gate"])
def test_every_operand_of_a_step_that_wants_a_gradient_is_refused(which):
    a = {k: torch.randn(4, 64, device="cuda") for k in ("x", "f", "h", "gate")}
    a["bias"] = torch.randn(64, device="cuda")
    a[which].requires_grad_()
    calls = [lambda kw=kw: recurrence.gated_scan_step(a["x"], a["f"], a["h"], bias=a["bias"], gate=a["gate"], **kw)
             for kw in ({}, {"inplace": True}, {"rows": torch.arange(4, dtype=torch.int32, device="cuda")})]
    for call in calls:
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
        with torch.no_grad():
            call()


def test_every_operand_of_an_8_bit_product_that_wants_a_gradient_is_refused():
    x, w = torch.randn(4, 64, device="cuda"), torch.randn(32, 64, device="cuda", requires_grad=True)
    (xq, xs), (wq, ws) = fp8.quantize(x), fp8.quantize_weight(w)  # weights are taken from parameters
    out = torch.empty(4, 32, device="cuda")
    on = lambda t: t.clone().requires_grad_()  # noqa: E731
    for call in (lambda: fp8.linear(on(x), wq, ws), lambda: fp8.linear(on(x), wq, ws, out=out),
                 lambda: fp8.linear(x, wq, on(ws)), lambda: fp8.linear(x, wq, on(ws), out=out),
                 lambda: fp8.quantize(on(x)), lambda: fp8.matmul(xq, on(xs), wq, ws),
                 lambda: fp8.matmul(xq, xs, wq, on(ws))):
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
        with torch.no_grad():
            call()


def test_8_bit_products_refuse_dual_operands():
    import torch.autograd.forward_ad as fwd
    x = torch.randn(4, 64, device="cuda")
    (xq, xs), (wq, ws) = fp8.quantize(x), fp8.quantize_weight(torch.randn(32, 64, device="cuda"))
    with fwd.dual_level(), torch.no_grad():
        a, s = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(ws, torch.ones_like(ws))
        for call in (lambda: fp8.quantize(a), lambda: fp8.linear(a, wq, ws, out=torch.empty(4, 32, device="cuda")),
                     lambda: fp8.linear(x, wq, s), lambda: fp8.matmul(xq, xs, wq, s)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        fp8.matmul(xq, xs, wq, ws)


def test_a_nan_row_does_not_end_a_generation():
    """A prompt that ends in NaN gives -1 from there on; the other rows are what they are without it."""
    m = _model().eval()
    with torch.no_grad():
        m.embed_tokens.weight[7] = float("nan")
    ids = torch.randint(8, 301, (4, 9), device="cuda")
    u = torch.rand(12, 4, device="cuda")
    kw = dict(max_new_tokens=12, temperature=0.9, top_k=30, top_p=0.95, uniforms=u)
    want = m.generate(ids, **kw)
    bad = ids.clone()
    bad[1, 4] = 7
    got = m.generate(bad, **kw)
    assert (got[1, 9:] == -1).all() and torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])
    assert ((want >= 0) & (want < 301)).all()


@pytest.mark.parametrize("use_fp8", [False, True])
def test_a_nan_row_does_not_end_a_decode_graph(use_fp8):
    m = _model(torch.bfloat16).eval()
    ids = torch.randint(301, (5, 17), device="cuda")
    settings = sampling.Sampler(temperature=0.8, top_k=40)
    with torch.no_grad():
        out = m(ids, return_states=True, last_logits_only=True)
        first = out["logits"][:, -1].argmax(-1)
        good = DecodeGraph(m, out["states"], first, sampler=settings, fp8=use_fp8)
        for (h,) in out["states"]:
            h[2] = float("nan")
        graph = DecodeGraph(m, out["states"], first, sampler=settings, fp8=use_fp8)
        rest = [0, 1, 3, 4]
        for _ in range(4):
            u = torch.rand(5, device="cuda")
            got, want = graph.step(u)[:, 0], good.step(u)[:, 0]
            assert got[2] == -1 and torch.isneginf(graph.logprobs[2])
            assert torch.equal(got[rest], want[rest]) and torch.equal(graph.logits[rest], good.logits[rest])


def test_a_decode_graph_reports_a_fault_at_the_next_step():
    """A replay's kernels record an expired wait in the fault word (written here by hand); step() raises it, once."""
    from prime_moment_attention_b200 import ops
    m = _model(torch.bfloat16).eval()
    ids = torch.randint(301, (2, 5), device="cuda")
    with torch.no_grad():
        out = m(ids, return_states=True, last_logits_only=True)
        graph = DecodeGraph(m, out["states"], out["logits"][:, -1].argmax(-1), fp8=True)
    graph.step()
    ops.check_faults(synchronize=True)
    ops._fault_view[0] = 131
    with pytest.raises(ops.KernelFault) as e:
        graph.step()
    assert e.value.code == 131
    graph.step()
