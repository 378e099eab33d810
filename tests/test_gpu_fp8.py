"""Block-scaled e4m3 quantisation and product against plain forms in float64.

Tolerances.  Quantisation is exact in its definition: e4m3(448 x / amax) with one float32 division;
the same expression in torch, tensor by tensor, gives the same bytes.  A product's terms are exact in
float32 (two 4-bit significands); a K block's sum of 128 of them and the sum over J blocks round by at most (128 + J)
2^-24 of the sum of magnitudes (any order; the tensor cores may truncate: 2^-23), and the scales'
product and the multiply by 3 2^-24 more: (300 + 2 J) 2^-23 of sum |x w| bounds a float32 result.
bf16 adds 2^-8 of the value.
"""
import pytest
import torch

from prime_moment_attention_b200 import _lib, fp8, ops

pytestmark = pytest.mark.gpu


def _pad(x, r, c):
    return torch.nn.functional.pad(x, (0, c - x.shape[1], 0, r - x.shape[0]))


def _over448(amax):
    """The correctly rounded quotient (torch divides by a number through its reciprocal)."""
    return (amax.double() / 448.0).float()


def _plain_rows(x):
    M, K = x.shape
    kb = -(-K // 128)
    g = _pad(x.float(), M, kb * 128).view(M, kb, 128)
    amax = g.abs().amax(2, keepdim=True).clamp_min(2.0 ** -100)
    return (g * 448.0 / amax).to(torch.float8_e4m3fn).view(M, -1)[:, :K], _over448(amax)[..., 0]


def _plain_blocks(w):
    N, K = w.shape
    nb, kb = -(-N // 128), -(-K // 128)
    g = _pad(w.float(), nb * 128, kb * 128).view(nb, 128, kb, 128)
    amax = g.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -100)
    q = (g * 448.0 / amax).to(torch.float8_e4m3fn).view(nb * 128, -1)[:N, :K]
    return q, _over448(amax)[:, 0, :, 0]


def _dequant(q, s, rows):
    K = q.shape[1]
    return q.double() * s.double().repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, :K]


def _data(M, N, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + M + 3 * N + 7 * K)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(1, K, generator=g))
    w = torch.randn(N, K, generator=g) / K ** 0.5 * torch.exp(torch.randn(N, 1, generator=g))
    return x.to(dtype).cuda(), w.to(dtype).cuda()


def _check_product(y, xq, xs, wq, ws):
    x, w = _dequant(xq, xs, 1), _dequant(wq, ws, 128)
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    J = -(-xq.shape[1] // 128)
    bar = (300 + 2 * J) * 2.0 ** -23 * mag + (2.0 ** -8 * want.abs() if y.dtype == torch.bfloat16 else 0.0)
    err = (y.double() - want).abs()
    assert (err <= bar).all(), (float((err / bar.clamp_min(1e-300)).max()), int((err > bar).sum()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (5, 128), (64, 768), (33, 1000), (300, 2050)])
def test_quantisation_is_bit_exact(M, K, dtype):
    x, w = _data(M, M, K, dtype)
    x[0] = 0                                     # an empty block
    x[-1] *= 1e-3
    if M > 2:
        x[1] = x[1] * 1e36 if dtype == torch.float32 else x[1] * 1e35
    q, s = fp8.quantize(x)
    pq, ps = _plain_rows(x)
    keep = x.float().abs().amax(1) < 1e35        # 448 x overflows in the plain form beyond
    assert torch.equal(q[keep].float(), pq[keep].float()) and torch.equal(s, ps)
    assert torch.isfinite(q.float()).all() and float(q.float().abs().max()) <= 448.0
    q, s = fp8.quantize_weight(w)
    pq, ps = _plain_blocks(w)
    assert torch.equal(q.float(), pq.float()) and torch.equal(s, ps)


SIZES = [(1, 1, 1), (1, 768, 2048), (2, 130, 128), (16, 128, 4096), (17, 100, 300), (32, 1000, 640), (50, 3000, 768),
         (64, 32000, 768), (65, 129, 257), (128, 128, 128), (129, 257, 1000), (200, 64, 5000), (777, 1530, 1000),
         (1024, 2048, 768), (2500, 2300, 512), (4096, 2560, 384), (8, 64, 8192),
         (256, 128, 4928), (130, 1000, 2111), (700, 300, 1100)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, out):
    x, w = _data(M, N, K, torch.bfloat16)
    (xq, xs), (wq, ws) = fp8.quantize(x), fp8.quantize_weight(w)
    _check_product(fp8.matmul(xq, xs, wq, ws, out_dtype=out), xq, xs, wq, ws)
    y = fp8.linear(x, wq, ws, out_dtype=out)
    _check_product(y, xq, xs, wq, ws)
    assert torch.equal(y, fp8.linear(x, wq, ws, out_dtype=out))  # repeats bit for bit


def test_layouts():
    """Scales and rows with other strides, outputs inside wider arrays, unaligned weights (copied)."""
    x, w = _data(70, 200, 500, torch.float32)
    (xq, xs), (wq, ws) = fp8.quantize(x), fp8.quantize_weight(w)
    want = fp8.matmul(xq, xs, wq, ws)
    assert torch.equal(want, fp8.matmul(xq, xs.contiguous(), wq, ws))
    wide = torch.zeros(70, 777, dtype=torch.bfloat16).cuda()
    fp8.matmul(xq, xs, wq, ws, out=wide[:, 5:205])
    assert torch.equal(wide[:, 5:205], want) and not wide[:, :5].any() and not wide[:, 205:].any()
    assert torch.equal(want, fp8.matmul(xq, xs, wq.contiguous(), ws))  # rows of 500 bytes
    assert torch.equal(want, fp8.matmul(xq, xs, wq, torch.cat([ws, ws], 1)[:, :4]))
    assert torch.equal(want, fp8.linear(x, wq, ws))
    cols = torch.zeros(70, 3 * 500).cuda()
    cols[:, 500:1000] = x
    assert torch.equal(want, fp8.linear(cols[:, 500:1000], wq, ws))
    assert torch.equal(want, fp8.linear(x.view(7, 10, 500), wq, ws).view(70, 200))
    assert torch.equal(want, fp8.linear(x.t().contiguous().t(), wq, ws))


def test_empty_and_nan():
    x, w = _data(4, 256, 256, torch.bfloat16)
    wq, ws = fp8.quantize_weight(w)
    assert fp8.linear(x[:0], wq, ws).shape == (0, 256)
    x[1, 130] = float("nan")
    x[2, 3] = float("inf")
    y = fp8.linear(x, wq, ws)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3]]).all()


def test_expired_wait_is_reported():
    x, w = _data(300, 256, 256, torch.bfloat16)
    wq, ws = fp8.quantize_weight(w)
    ops.check_faults(synchronize=True)
    for m in (300, 8):
        _lib.load().pma_test_expire_waits(1_000_000)
        try:
            fp8.linear(x[:m], wq, ws)
        finally:
            _lib.load().pma_test_expire_waits(0)
        torch.cuda.synchronize()
        with pytest.raises(ops.KernelFault) as e:
            fp8.linear(x[:m], wq, ws)
        assert e.value.code == 130
        fp8.linear(x[:m], wq, ws)
        ops.check_faults(synchronize=True)


def test_expired_wait_on_pairs_is_reported():
    x, w = _data(2560, 2304, 256, torch.bfloat16)
    wq, ws = fp8.quantize_weight(w)
    ops.check_faults(synchronize=True)
    _lib.load().pma_test_expire_waits(1_000_000)
    try:
        fp8.linear(x, wq, ws)
    finally:
        _lib.load().pma_test_expire_waits(0)
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelFault) as e:
        fp8.linear(x, wq, ws)
    assert e.value.code == 130
    fp8.linear(x, wq, ws)
    ops.check_faults(synchronize=True)


def test_offsets_past_32_bits():
    """x of more than 2^31 elements and y of more than 2^32 bytes: the last rows as a call of their own
    gives them."""
    M, K, N = 270000, 8192, 8192
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda").normal_()
    wq, ws = fp8.quantize_weight(torch.randn(N, K, device="cuda"))
    y = fp8.linear(x, wq, ws)
    tail = slice(M - 256, M)  # other tiles than the long call's: equal to the order of the sums
    torch.testing.assert_close(y[tail].float(), fp8.linear(x[tail], wq, ws).float(), rtol=2.0 ** -7, atol=1e-2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("exponent", [-100, -7, 0, 90])
def test_every_quotient_of_bf16_values(dtype, exponent):
    """Each pair of an 8-bit significand and an 8-bit largest one, x from amax down to where it rounds to
    zero, both signs: the bytes of the quotient in 64 bits. (Float32 on the way to e4m3 is harmless: a
    quotient that is not midway between two e4m3 values is 2^-13 of its size from there.)"""
    a = torch.arange(128, 256, dtype=torch.float64)[:, None, None, None]
    down = torch.arange(0, 22, dtype=torch.float64)[None, :, None, None]
    sign = torch.tensor([1.0, -1.0], dtype=torch.float64)[None, None, :, None]
    mant = torch.cat([torch.arange(128, 255), torch.arange(129, 256)]).to(torch.float64)
    x = torch.minimum(mant * 2.0 ** -down, a) * sign                       # (128, 22, 2, 254)
    lead = a.expand(128, 22, 2, 1)
    x = torch.cat([lead, x[..., :127], lead, x[..., 127:]], -1).reshape(-1, 256) * 2.0 ** (exponent - 7)
    amax = (a * 2.0 ** (exponent - 7)).expand(128, 22, 2, 1).reshape(-1, 1)
    want = (448 * x / amax).float().to(torch.float8_e4m3fn).view(torch.uint8)
    xq, xs = fp8.quantize(x.to(dtype).cuda())
    assert torch.equal(xq.view(torch.uint8).cpu(), want)
    torch.testing.assert_close(xs[:, 0].double().cpu(), amax[:, 0] / 448, rtol=2.0 ** -23, atol=0)


@pytest.mark.parametrize("M,N,K", [(70, 300, 500), (8, 300, 500), (300, 520, 100), (3, 300, 100), (2600, 2304, 256), (5, 100, 300)])
def test_scales_of_any_strides(M, N, K):
    """Scales that are a broadcast (one row for all, one number for all), overlapping, transposed or strided views give
    what the same numbers give as an array of their own."""
    x, w = _data(M, N, K, torch.bfloat16)
    (xq, xs), (wq, _) = fp8.quantize(x), fp8.quantize_weight(w)
    nb, kb = -(-N // 128), -(-K // 128)
    g = torch.Generator().manual_seed(5)
    v = (torch.rand(4 * nb * kb, generator=g) + 0.5).cuda()
    views = [v[:kb].expand(nb, kb), v[:nb, None].expand(nb, kb), v[:1].expand(nb, kb), v.as_strided((nb, kb), (1, 1)),
             v.as_strided((nb, kb), (1, nb)), v.as_strided((nb, kb), (2 * kb, 2)), v.as_strided((nb, kb), (kb + 1, 1))]
    for ws in views:
        dense = ws.clone(memory_format=torch.contiguous_format)
        assert torch.equal(fp8.matmul(xq, xs, wq, ws), fp8.matmul(xq, xs, wq, dense))
        assert torch.equal(fp8.linear(x, wq, ws), fp8.linear(x, wq, dense))
        _check_product(fp8.linear(x, wq, ws, out_dtype=torch.float32), xq, xs, wq, dense)
    for one in (xs[:1].expand(M, kb), xs[:, :1].expand(M, kb)):  # and those of x
        _check_product(fp8.matmul(xq, one, wq, dense), xq, one, wq, dense)


def test_float32_ties_go_by_the_float32_quotient():
    """Float32 values whose exact quotient lies half-way between two e4m3 values, and their neighbours: the bytes of the
    float32 expression, and never farther from x than half a step of e4m3 (2^-4 of a binade) and the two
    roundings, 2^-23 of the value."""
    g = torch.Generator().manual_seed(3)
    n = 4096
    m = torch.randint(1 << 18, 1 << 19, (n, 1), generator=g).double()       # 448 (m t) / (7 m) = 64 t
    t = torch.randint(8, 16, (n, 40), generator=g).double() * 2 + 1          # between two significands of 4 bits
    x = (m * t * 2.0 ** torch.randint(-13, -2, (n, 40), generator=g).double()).float()  # 24 bits: 448 x has more
    amax, none = (7 * m).float(), torch.zeros(())
    both = torch.cat([amax, x, x.nextafter(none), x.nextafter(none + 1e9)], 1)
    both = torch.cat([both, torch.tensor([[2089626.0, 79293.84375] + [0.0] * (both.shape[1] - 2)])]).cuda()
    q, s = fp8.quantize(both)
    pq, ps = _plain_rows(both)
    assert torch.equal(q.view(torch.uint8), pq.view(torch.uint8)) and torch.equal(s, ps)
    back = q.double() * both.double().amax(1, keepdim=True) / 448
    v = both.double() * 448 / both.double().amax(1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 3)
    assert ((back - both.double()).abs() * 448 / both.double().amax(1, keepdim=True) <= step / 2 + 2.0 ** -23 * v).all()
