"""The token sampler against the rule in float64 (tests/sampling_oracle.py).

A float32 weight is within d = 3e-7 (relative) of exp(z) for the z here that matter (z > -23: the
product rounds z by 2^-24 |z| < 1.4e-6 at most at its far end, where weights are below 1e-9 of the
largest; at the near end, |z| < 2, by 1.2e-7, plus 1.2e-7 of the exponential) and rounding to 2^-32
adds V 2^-33 in all.  So an edge of a token's interval is off by at most EDGE = 1e-6 + V 2^-33 of the
kept weight, and the token is checked by its interval.  A cut may move by as much: the interval is
taken over every set that a cut within EDGE leaves.
"""
import numpy as np
import pytest
import torch

from prime_moment_attention_b200 import sampling
from tests import sampling_oracle as O

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _per_row(v, i):
    return v[i].item() if isinstance(v, torch.Tensor) else v


def _check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    tok, lp = sampling.sample(logits, u, temperature, top_k, top_p, min_p)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    x, tok, lp, u = logits.float().cpu().numpy(), tok.cpu().numpy(), lp.cpu().numpy(), u.cpu().double().numpy()
    B, V = x.shape
    edge = 1e-6 + V * 2.0 ** -33
    for b in range(B):
        T, k, p, m = (_per_row(v, b) for v in (temperature, top_k, top_p, min_p))
        idx, _, logz, z = O.row(x[b], T, k, p, m)
        if len(idx) == 0:
            assert tok[b] == -1 and lp[b] == -np.inf
            continue
        # the kept set with every cut moved by the weights' error either way: whichever of them the
        # kernel cut, its token's interval lies between these ends
        e = np.exp(z)
        lo = O.row(x[b], T, k, p - edge if p < 1 else p, m * (1 + 1e-6))[0]
        hi = O.row(x[b], T, k, min(p + edge, 1.0) if p < 1 else p, m * (1 - 1e-6))[0]
        assert tok[b] in hi, (b, tok[b], "not kept")
        begin = e[lo[lo < tok[b]]].sum() / e[hi].sum()
        end = e[hi[hi <= tok[b]]].sum() / e[lo].sum()
        assert begin - edge <= u[b] <= end + edge, (b, tok[b], begin, u[b], end)
        assert abs(lp[b] - (z[tok[b]] - logz)) <= 2e-6 * max(1.0, abs(z[tok[b]]), abs(logz)) + V * 2.0 ** -33
    return tok


def _logits(B, V, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * scale
    x[:, : max(1, V // 50)] += 4.0
    x = x[:, torch.randperm(V, generator=g)]
    return x.to(DT[dtype]).cuda(), torch.rand(B, generator=g).cuda()


SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=50), dict(top_k=700), dict(top_p=0.9),
            dict(top_p=0.3, temperature=1.4), dict(min_p=0.05), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.01),
            dict(top_k=9000, top_p=0.99, temperature=1.2)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 33, 1000, 5003, 32000, 131072])
@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "plain")
def test_tokens_and_logprobs(dtype, V, kw):
    x, u = _logits(5, V, dtype, seed=V)
    _check(x, u, **kw)


@pytest.mark.parametrize("B,V", [(300, 4096), (149, 8191), (2, 360448)])
def test_batches_with_settings_per_row(B, V):
    x, u = _logits(B, V, "f32", seed=B)
    g = torch.Generator().manual_seed(1)
    pick = lambda vals, dt: torch.tensor(vals, dtype=dt)[torch.randint(len(vals), (B,), generator=g)].cuda()  # noqa: E731
    kw = dict(temperature=pick([0.0, 0.5, 1.0, 1.7], torch.float32), top_k=pick([0, 1, 7, 300, V + 5], torch.int32),
              top_p=pick([1.0, 0.95, 0.5, 0.0], torch.float32), min_p=pick([0.0, 0.1, 2.0], torch.float32))
    tok = _check(x, u, **kw)
    # a row alone, with its settings, gives the token it gave in the batch
    for b in range(0, B, max(1, B // 7)):
        one = sampling.sample(x[b:b + 1], u[b:b + 1], *(v[b].item() for v in kw.values()))[0]
        assert one.item() == tok[b]


def test_the_ends_of_the_draw():
    x, _ = _logits(4, 999, "f32")
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, float("nan")]).cuda()
    tok = sampling.sample(x, u)[0].cpu().numpy()
    assert tok[0] == 0 and tok[3] == 0        # the first token with weight
    assert tok[1] == 998 and tok[2] == 998    # the last one; u = 1 is clamped into the row


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [64, 40000])
def test_equal_logits_go_by_index(dtype, V):
    """All logits equal: top-k keeps the first k indices, top-p the first ceil(p V); the token is
    floor(u n) of the n kept."""
    x = torch.full((3, V), 1.5, dtype=DT[dtype]).cuda()
    u = torch.tensor([0.0, 0.5, 0.999]).cuda()
    assert sampling.sample(x, u, temperature=0.0)[0].tolist() == [0, 0, 0]
    assert sampling.sample(x, u, top_k=10)[0].tolist() == [0, 5, 9]
    n = V // 4
    want = [0, n // 2, int(float(u[2].item()) * n)]
    assert sampling.sample(x, u, top_p=0.25)[0].tolist() == want
    assert sampling.sample(x, u, top_k=V - 1, top_p=0.25)[0].tolist()[:2] == [0, (n - (n > 0) + 1) // 2]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_few_distinct_values(dtype):
    """Ties across every cut: logits take 5 values, cuts fall inside a value."""
    g = torch.Generator().manual_seed(2)
    x = torch.tensor([0.0, -1.0, -2.0, -0.0, 1.0])[torch.randint(5, (6, 20011), generator=g)].to(DT[dtype]).cuda()
    u = torch.rand(6, generator=g).cuda()
    for k in (1, 10, 4000, 4100, 12345, 20000):
        _check(x, u, top_k=k)
    for p in (0.1, 0.6, 0.97):
        _check(x, u, top_p=p)


def test_masked_rows():
    x, u = _logits(6, 3001, "f32", seed=5)
    x[0] = -float("inf")                        # nothing left
    x[1] = float("nan")                         # nothing left
    x[2, 1:] = -float("inf")                    # one token
    x[3, ::2] = float("nan")                    # half of the row
    x[4, 100] = x[4, 200] = float("inf")        # two tokens share the row
    x[5] = torch.finfo(torch.float32).min       # a mask of the lowest value is a logit like another
    for kw in (dict(), dict(top_k=20), dict(top_p=0.8), dict(temperature=0.0), dict(min_p=0.1, top_k=3)):
        tok = sampling.sample(x, u, **kw)[0].tolist()
        assert tok[0] == -1 and tok[1] == -1 and tok[2] == 0 and tok[3] % 2 == 1 and tok[4] in (100, 200)
        assert 0 <= tok[5] < 3001
        _check(x[2:4], u[2:4], **kw)
    lp = sampling.sample(x, u)[1]
    assert torch.isneginf(lp[:2]).all() and lp[2] == 0.0
    assert abs(lp[4].item() + np.log(2.0)) < 1e-6
    assert abs(lp[5].item() + np.log(3001.0)) < 2e-5


def test_strided_rows_and_unaligned_starts():
    x, u = _logits(7, 5000, "bf16", seed=9)
    wide = torch.zeros(7, 5011, dtype=torch.bfloat16).cuda()
    wide[:, 3:5003] = x
    for kw in (dict(top_p=0.9), dict(top_k=30)):
        a, b = sampling.sample(x, u, **kw), sampling.sample(wide[:, 3:5003], u, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = x.t().contiguous().t()  # columns contiguous: copied
    assert torch.equal(sampling.sample(t, u)[0], sampling.sample(x, u)[0])


def test_frequencies_follow_the_distribution():
    """Counts over 40,000 evenly spaced u against the probabilities: the inverse transform of an even
    grid is within one grid step of them."""
    x = torch.tensor([[0.0, 1.0, 2.0, 3.0, -float("inf"), 2.5]]).cuda()
    n = 40000
    u = ((torch.arange(n) + 0.5) / n).float().cuda()
    tok = sampling.sample(x.expand(n, 6), u)[0]
    got = torch.bincount(tok, minlength=6).double() / n
    want = torch.softmax(x[0].double(), 0)
    assert (got - want.cuda()).abs().max() < 2.0 / n


def test_greedy_in_a_graph():
    x, u = _logits(8, 32000, "bf16", seed=11)
    want = sampling.sample(x, u, top_k=50)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sampling.sample(x, u, top_k=50)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = sampling.sample(x, u, top_k=50)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_empty_batch():
    tok, lp = sampling.sample(torch.zeros(0, 10).cuda(), torch.zeros(0).cuda())
    assert tok.shape == (0,) and lp.shape == (0,)


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last rows as a call of their own gives them."""
    B, V = 17000, 131072
    x = torch.empty(B, V, dtype=torch.bfloat16, device="cuda").normal_().mul_(3)
    u = torch.rand(B, device="cuda")
    tok, lp = sampling.sample(x, u, top_k=50, top_p=0.9)
    for b in (0, 16383, 16384, 16999):
        one = sampling.sample(x[b:b + 1], u[b:b + 1], top_k=50, top_p=0.9)
        assert one[0] == tok[b] and one[1] == lp[b]
