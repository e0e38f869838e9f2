"""The 4-bit key / value cache: write, read back, attention over it; CPU and CUDA."""

import math
from fractions import Fraction

import pytest
import torch

from underhfs.kv_cache import RANGE, QuantizedKVCache, quantize_groups

H16 = torch.finfo(torch.float16).eps / 2  # one rounding to fp16, relative


def attention(q, k, v, pos, window, sinks, scale):
    """q [T, H, D], k / v [n, H, D] in 64 bits, pos [T]: (o, sum p |v|, sum |q||k| of the largest score)."""
    s = torch.einsum("thd,nhd->htn", q, k) * scale
    size = torch.einsum("thd,nhd->htn", q.abs(), k.abs()) * scale
    j = torch.arange(k.shape[0], device=q.device)
    ok = j[None, :] <= pos[:, None]
    if window:
        ok &= (pos[:, None] - j[None, :] < window) | (j[None, :] < sinks)
    s = s.masked_fill(~ok, float("-inf"))
    p = torch.softmax(s, -1)
    size = size.masked_fill(~ok, 0).amax(-1)
    return (torch.einsum("htn,nhd->thd", p, v), torch.einsum("htn,nhd->thd", p, v.abs()), size.transpose(0, 1))


# ------------------------------------------------------------------- CPU
def test_quantised_values_are_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 96, generator=g) * torch.logspace(-3, 3, 50).unsqueeze(1) + 5
    y = quantize_groups(x)
    w = x.double().unflatten(-1, (-1, 32))
    lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
    # half a step, and what the fp16 roundings of the minimum and of 15 steps can leave uncovered
    bound = (hi - lo) / 30 * (1 + 2 * H16) + H16 * lo.abs() + H16 * (hi - lo) + 2.0**-24
    assert ((y.unflatten(-1, (-1, 32)) - w).abs() <= bound).all()
    assert (y.unflatten(-1, (-1, 32)) - w).abs().max() > 0
    for i in range(3):
        assert len(torch.unique(y[0, i * 32 : i * 32 + 32])) <= 16


def test_quantised_special_values():
    nan, inf = float("nan"), float("inf")
    x = torch.zeros(6, 32)
    x[1] = 3.0
    x[2, :3] = torch.tensor([inf, -inf, 1e30])
    x[3, :2] = torch.tensor([nan, 7.0])
    x[4] = nan
    x[5] = 1e-9
    y = quantize_groups(x)
    assert torch.isfinite(y).all() and y.abs().max() <= RANGE * (1 + 2 * H16)
    assert (y[0] == 0).all() and (y[1] == 3).all() and (y[4] == 0).all()
    assert y[2, 0] == y[2, 2] == RANGE and y[2, 1] == -RANGE
    assert y[3, 0] == 0 and abs(y[3, 1] - 7) < 15 * 7 * H16


def format_by_fractions(x):
    """The documented format in exact arithmetic, group by group: lo = fp16(min), s = fp16(fp32(fp32(max - lo) *
    fp32(1 / 15))), code = (x - lo) / s rounded half to even, held to 0..15."""
    import numpy as np

    def near(v):  # half to even
        k = v.numerator // v.denominator
        rest = v - k
        return k + (rest > Fraction(1, 2) or (rest == Fraction(1, 2) and k % 2))

    out = []
    for row in x.reshape(-1, 32).float().numpy():
        lo = np.float16(row.min())
        s = np.float16(np.float32(row.max() - np.float32(lo)) * np.float32(1 / 15))
        lo, s = Fraction(float(lo)), Fraction(float(s))
        out.append([float(lo + s * max(0, min(15, near((Fraction(float(v)) - lo) / s) if s else 0))) for v in row])
    return torch.tensor(out, dtype=torch.float64).view(x.shape)


def format_inputs(dtype):
    g = torch.Generator().manual_seed(11)
    x = torch.randn(6, 40, 64, generator=g)
    x[1] = x[1] * 1e-3 + 0.7
    x[2] *= torch.logspace(-4, 4, 40).unsqueeze(1)
    x[3] = (x[3] * 8).round() / 4
    x[4] = torch.randint(0, 31, (40, 64), generator=g) * 0.5  # quotients on halves
    x[5] = torch.randint(-3, 4, (40, 64), generator=g).float() * 1000
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantised_values_are_those_of_the_format(dtype):
    x = format_inputs(dtype)
    assert torch.equal(quantize_groups(x), format_by_fractions(x))


def test_cpu_cache_holds_and_attends():
    torch.manual_seed(1)
    cache = QuantizedKVCache(2, 2, 2, 32, 12, device="cpu")
    k, v = torch.randn(2, 5, 2, 32), torch.randn(2, 5, 2, 32)
    cache.append(1, k, v, counts=torch.tensor([5, 3]))
    cache.advance(torch.tensor([4, 3]))
    kk, vv = cache.read(1, 0, 6, dtype=torch.float64)
    assert torch.equal(kk[0, :5], quantize_groups(k[0])) and torch.equal(vv[1, :3], quantize_groups(v[1, :3]))
    assert (kk[1, 3:] == 0).all() and (cache.read(0)[0] == 0).all()
    cache.append(1, k[:, :2] + 1, v[:, :2] + 1)  # sequence 0 writes over its token 4
    assert torch.equal(cache.read(1, 4, 2, dtype=torch.float64)[0][0], quantize_groups(k[0, :2] + 1))
    q = torch.randn(2, 2, 4, 32, dtype=torch.float64)
    for window, sinks in ((None, 0), (2, 1)):
        o = cache.attend(1, q, window=window, sinks=sinks)
        kk, vv = (t.repeat_interleave(2, 2) for t in cache.read(1, dtype=torch.float64))
        for b, start in ((0, 4), (1, 3)):
            n = start + 2
            want, _, _ = attention(q[b], kk[b, :n], vv[b, :n], torch.arange(start, n), window, sinks, 32**-0.5)
            assert torch.allclose(o[b], want, rtol=0, atol=1e-12)
    assert (cache.attend(1, q, counts=torch.tensor([2, 1]))[1, 1] == 0).all()


def test_refusals_on_the_cpu():
    with pytest.raises(ValueError, match="head_dim"):
        QuantizedKVCache(1, 1, 1, 40, 8, device="cpu")
    with pytest.raises(ValueError, match="max_len"):
        QuantizedKVCache(1, 1, 1, 32, 0, device="cpu")
    c = QuantizedKVCache(1, 2, 2, 32, 8, device="cpu")
    x = torch.zeros(2, 3, 2, 32)
    with pytest.raises(IndexError):
        c.append(1, x, x)
    with pytest.raises(ValueError, match="k must be"):
        c.append(0, x[:1], x[:1])
    with pytest.raises(ValueError, match="differ"):
        c.append(0, x, x.double())
    with pytest.raises(ValueError, match="counts"):
        c.append(0, x, x, counts=torch.ones(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="counts"):
        c.append(0, x, x, counts=torch.ones(2))
    with pytest.raises(TypeError, match="floating"):
        c.append(0, x.long(), x.long())
    with pytest.raises(ValueError, match="multiple"):
        c.attend(0, torch.zeros(2, 1, 3, 32))
    for bad in (dict(window=0), dict(sinks=2), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            c.attend(0, torch.zeros(2, 1, 2, 32), **bad)
    c.append(0, x, x)
    c.advance(3)
    c.append(0, x, x)
    c.advance(3)
    for call in (lambda: c.append(0, x, x), lambda: c.attend(0, x), lambda: c.advance(3),
                 lambda: c.append(0, x, x, counts=torch.tensor([1, 3]))):
        with pytest.raises(ValueError, match="do not fit"):
            call()
    with pytest.raises(ValueError, match="outside"):
        c.read(0, 7, 2)
    c.reset()
    c.append(0, x, x)


# ------------------------------------------------------------------- GPU
@pytest.fixture
def status():
    from underhfs_b200.ops._lib import core

    yield lambda: core().device_status(True)
    st = core().device_status(True)
    assert st["code"] == 0, st


def randn(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,D", [(1, 1, 64), (2, 3, 128), (3, 5, 64)])
def test_written_and_read_back(B, H, D, dtype, status):
    """Appends of many lengths, page borders crossed; the values are the format's, bit for bit."""
    cache = QuantizedKVCache(2, B, H, D, 150)
    want = torch.zeros(2, B, 150, H, D, dtype=torch.float64, device="cuda")
    at = 0
    for n, t in enumerate((1, 30, 1, 1, 33, 64, 2)):
        k = 3 * randn(B, t, H, D, seed=n, dtype=dtype) + 1
        v = randn(B, t, H, D, seed=100 + n, dtype=dtype)
        cache.append(1, k, v)
        cache.advance(t)
        want[0, :, at : at + t], want[1, :, at : at + t] = quantize_groups(k), quantize_groups(v)
        at += t
    assert cache.lengths.tolist() == [at] * B
    for out in (torch.float32, torch.bfloat16, torch.float16):
        for got, x in zip(cache.read(1, dtype=out), want):
            assert torch.equal(got, x.float().to(out))
        for got, x in zip(cache.read(1, 29, 70, dtype=out), want):
            assert torch.equal(got, x[:, 29:99].float().to(out))
    assert all((t == 0).all() for t in cache.read(0))


@pytest.mark.gpu
def test_written_from_strided_rows_and_ragged_batches(status):
    B, T, H, D = 3, 45, 2, 64
    qkv = randn(B * T, 3 * H * D, seed=5)
    _, k, v = qkv.view(B, T, 3, H, D).unbind(2)  # fused projection, as the engine has it
    kt = randn(B, H, T, D, seed=6).transpose(1, 2)  # heads first
    odd = randn(B * T * H * D + 1, seed=7)[1:].view(B, T, H, D)  # not 16-byte aligned
    wide = randn(B, T, H, 2 * D, seed=8)[..., ::2]  # channels apart
    counts = torch.tensor([45, 0, 17], dtype=torch.int32, device="cuda")
    for a, b in ((k, v), (kt, odd), (wide, k)):
        cache = QuantizedKVCache(1, B, H, D, 64)
        old_k, old_v = randn(B, 64, H, D, seed=9), randn(B, 64, H, D, seed=10)
        cache.append(0, old_k, old_v)
        cache.advance(3)
        cache.append(0, a, b, counts=counts)
        for got, new, old in zip(cache.read(0, dtype=torch.float32), (a, b), (old_k, old_v)):
            want = quantize_groups(old)
            for s, n in enumerate(counts.tolist()):
                want[s, 3 : 3 + n] = quantize_groups(new[s, :n])
            assert torch.equal(got, want.float())  # and what was not written is as it was


@pytest.mark.gpu
def test_special_values_are_stored_finite(status):
    nan, inf = float("nan"), float("inf")
    x = torch.zeros(1, 8, 1, 64, device="cuda")
    x[0, 1] = 3.0
    x[0, 2, 0, :4] = torch.tensor([inf, -inf, 1e30, nan], device="cuda")
    x[0, 3] = nan
    x[0, 4] = 1e-9
    x[0, 5] = torch.linspace(-1e-6, 1e-6, 64)
    x[0, 6] = torch.linspace(61439, 61440, 64)
    x[0, 7] = torch.arange(64) * 0.25  # quotients on halves
    for dtype in (torch.float32, torch.bfloat16):
        cache = QuantizedKVCache(1, 1, 1, 64, 8)
        cache.append(0, x.to(dtype), x.to(dtype))
        for got in cache.read(0, dtype=torch.float32):
            assert torch.equal(got, quantize_groups(x.to(dtype)).float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_stored_values_are_those_of_the_format(dtype, status):
    x = format_inputs(dtype)
    cache = QuantizedKVCache(1, 6, 1, 64, 40)
    cache.append(0, x.unsqueeze(2).cuda(), -x.unsqueeze(2).cuda())
    for got, want in zip(cache.read(0, dtype=torch.float32), (x, -x)):
        assert torch.equal(got[:, :, 0].double().cpu(), format_by_fractions(want).float().double())


def fill(B, keys, Hkv, D, lens, tq, dtype, seed=0):
    """A cache whose sequence b holds lens[b] tokens, the last tq of them not yet advanced."""
    cache = QuantizedKVCache(1, B, Hkv, D, keys)
    k = randn(B, keys, Hkv, D, seed=seed, dtype=dtype) + randn(1, 1, Hkv, D, seed=seed + 1, dtype=dtype)
    v = randn(B, keys, Hkv, D, seed=seed + 2, dtype=dtype)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cache.append(0, k, v, counts=n)
    cache.advance(n - torch.tensor(tq, dtype=torch.int32, device="cuda"))
    return cache


def check_attend(cache, q, got, lens, tq, window, sinks, scale=None):
    """Against 64 bits over the cached values.

    q and the codes go in exactly (q may lose what is 2^-25 of its largest element: a score
    moves by that times sum|k|), the fp32 sums of a score by a few 2^-23 of sum|q| (|lo| + 15 s).
    Of v, P s and lo + 8 s are rounded to fp16 (H16), the first for s (code - 8), |code - 8| <= 8;
    below fp16's normal range P s is off by 2^-25, for at most 8 steps.  Then the result's rounding.
    """
    D, G = q.shape[3], q.shape[2] // cache.kv_heads
    scale = D**-0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    kk, vv = (t.double().repeat_interleave(G, 2) for t in cache.read(0, dtype=torch.float32))
    # 8 s + |lo + 8 s| of each value's group: codes 0 and 15 are both in it
    g = vv.unflatten(-1, (-1, 32))
    lo, step = g.amin(-1, keepdim=True), (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) / 15
    part = (8 * step + (lo + 8 * step).abs()).expand(g.shape).flatten(-2)
    for b, (n, t) in enumerate(zip(lens, tq)):
        assert (got[b, t:] == 0).all()
        if t == 0:
            continue
        pos = torch.arange(n - t, n, device="cuda")
        qb = q[b, :t].double()
        o, _, score = attention(qb, kk[b, :n], vv[b, :n], pos, window, sinks, scale)
        size, rounded = (attention(qb, kk[b, :n], x[b, :n], pos, window, sinks, scale)[0] for x in (vv.abs(), part))
        big = scale * kk[b, :n].abs().max() * q.shape[3] * qb.abs().amax(-1)
        move = 2.0**-25 * big + 2.0**-20 * (score + big)
        err = torch.expm1(2 * move).unsqueeze(-1) * size + H16 * rounded + half * o.abs()
        err = 1.01 * err + n * 2.0**-22 + 1e-6
        over = ((got[b, :t].double() - o).abs() - err).max().item()
        assert over <= 0, (b, over)


CASES = [  # B, tq, lens, Hq, Hkv, D, window, sinks
    (1, [1], [1], 1, 1, 64, None, 0),
    (2, [1, 1], [2, 31], 3, 3, 128, None, 0),
    (4, [1, 1, 1, 1], [32, 33, 64, 65], 2, 2, 64, None, 0),
    (1, [1], [1000], 12, 12, 64, None, 0),
    (1, [1], [3001], 2, 1, 128, None, 0),
    (3, [1, 0, 1], [700, 300, 1], 8, 1, 128, None, 0),
    (2, [40, 13], [40, 13], 2, 2, 64, None, 0),
    (2, [5, 5], [500, 77], 8, 1, 128, None, 0),
    (2, [9, 4], [333, 96], 6, 2, 64, None, 0),
    (2, [1, 1], [500, 20], 4, 2, 64, 33, 1),
    (2, [1, 1], [640, 641], 4, 4, 128, 1, 0),
    (1, [17], [900], 4, 2, 128, 100, 40),
    (1, [60], [200], 1, 1, 64, 7, 3),
    (2, [3, 3], [4000, 90], 5, 1, 64, 64, 200),
    (1, [2], [2048], 24, 1, 128, 2047, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,tq,lens,Hq,Hkv,D,window,sinks", CASES)
def test_attention(B, tq, lens, Hq, Hkv, D, window, sinks, dtype, status):
    cache = fill(B, max(lens) + 3, Hkv, D, lens, tq, dtype)
    q = randn(B, max(tq), Hq, D, seed=50, dtype=dtype)
    counts = torch.tensor(tq, dtype=torch.int32, device="cuda") if len(set(tq)) > 1 else None
    got = cache.attend(0, q, window=window, sinks=sinks, counts=counts)
    check_attend(cache, q, got, lens, tq, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 5)])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (6, 2, 128)])
def test_attention_of_prompts_onto_a_filled_cache(Hq, Hkv, D, window, sinks, status):
    """Hundreds of new tokens (many tiles of queries to a head) behind cached ones, ragged."""
    lens, tq = [1500, 700], [601, 300]
    cache = fill(2, 1600, Hkv, D, lens, tq, torch.bfloat16)
    q = randn(2, 601, Hq, D, seed=57)
    counts = torch.tensor(tq, dtype=torch.int32, device="cuda")
    check_attend(cache, q, cache.attend(0, q, window=window, sinks=sinks, counts=counts), lens, tq, window, sinks)


@pytest.mark.gpu
def test_attention_strides_scale_and_large_queries(status):
    lens, tq = [300, 41], [2, 2]
    cache = fill(2, 320, 2, 64, lens, tq, torch.bfloat16)
    qkv = randn(2 * 2, 3 * 4 * 64, seed=51).view(2, 2, 3, 4, 64)
    odd = randn(2 * 2 * 4 * 64 + 3, seed=52)[3:].view(2, 2, 4, 64)
    for q in (qkv[:, :, 1], odd, randn(2, 4, 2, 64, seed=53).transpose(1, 2)):
        check_attend(cache, q, cache.attend(0, q, scale=0.3), lens, tq, None, 0, 0.3)
    # the power of two that brings q to fp16's range: results as for q of ordinary size
    big = randn(2, 2, 4, 64, seed=54)
    a = cache.attend(0, big, scale=0.125)
    assert torch.equal(a, cache.attend(0, big * 2.0**60, scale=0.125 * 2.0**-60))
    assert torch.equal(a, cache.attend(0, big * 2.0**-40, scale=0.125 * 2.0**40))
    assert (cache.attend(0, torch.zeros_like(big)).isfinite()).all()
    big[0, 0, 1, 5] = float("nan")
    got = cache.attend(0, big, scale=0.125)
    assert got[0, 0, 1].isnan().all()
    got[0, 0, 1], a[0, 0, 1] = 0, 0
    assert torch.equal(got, a)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,size", [(4096, 1.0), (4096, 1e-2), (4096, 1e-4), (32768, 1e-3), (32768, 1e-4), (32768, 30.0)])
def test_attention_keeps_small_and_large_values(n, size, D, status):
    """Long contexts whose probabilities span many powers of two (scores of standard deviation 2.5), with
    values of any size: the error is that of the roundings, not of fp16's range.

    In the 2-norm over thousands of outputs, independent roundings add by their squares: of each token
    P s (8 steps at most) and lo + 8 s, H16 of themselves or 2^-25 where they are below fp16's normal range;
    P s enters as at least 2^10 times itself, P at least its ratio to the largest: its 2^-25 is
    2^-35 of the largest probability.  Twice that, and the result's own rounding.  (40 sequences: a
    warp has an eighth of the keys, and one maximum for them.)"""
    B, Hkv, G = 40, 4, 2
    cache = QuantizedKVCache(1, B, Hkv, D, n)
    k, v = randn(1, n, Hkv, D, seed=1), (size * randn(1, n, Hkv, D, seed=2).float()).bfloat16()
    cache.append(0, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1))
    cache.advance(n - 1)
    q = (2.5 * randn(B, 1, Hkv * G, D, seed=3).float()).bfloat16()
    got = cache.attend(0, q)[:, 0].double().view(B, Hkv, G, D)
    kk, vv = (t[0].double() for t in cache.read(0, dtype=torch.float32))
    p = torch.softmax(torch.einsum("bhgd,nhd->bhgn", q.double().view(B, Hkv, G, D), kk) * D**-0.5, -1)
    o = torch.einsum("bhgn,nhd->bhgd", p, vv)
    g = vv.unflatten(-1, (-1, 32))
    lo, step = g.amin(-1, keepdim=True), (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) / 15
    mid = (lo + 8 * step).abs()
    part = ((H16 * 8 * step) ** 2 + torch.maximum(H16 * mid, torch.full_like(mid, 2.0**-25)) ** 2).expand(g.shape).flatten(-2)
    small = (8 * 2.0**-35 * n**0.5 * p.amax(-1)).norm() * D**0.5
    spread = torch.einsum("bhgn,nhd->bhgd", p**2, part).sqrt().norm() + small
    assert (got - o).norm() <= torch.finfo(torch.bfloat16).eps / 2 * o.norm() + 2 * spread


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_over_values_of_all_sizes_at_once(D, dtype, status):
    """Tokens of ordinary values, then some thousands of times larger (to the format's range), then ordinary
    ones: nothing overflows, and a query that does not see the large ones has the bits it has without them."""
    lens, tq = [900, 700], [6, 6]
    q = randn(2, 6, 4, D, seed=60, dtype=dtype)
    outs = []
    for large in (1.0, 100.0, 3000.0, RANGE / 5):
        cache = QuantizedKVCache(1, 2, 2, D, 900)
        k, v = randn(2, 900, 2, D, seed=61, dtype=dtype), randn(2, 900, 2, D, seed=62, dtype=dtype)
        for at in (5, 211, 450, 691, 897):  # (the last two are seen by some of the new tokens only)
            v[:, at] = (large * v[:, at].float()).to(dtype)
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cache.append(0, k, v, counts=n)
        cache.advance(n - 6)
        for window in (None, 400):
            got = cache.attend(0, q, window=window)
            assert got.isfinite().all()
            check_attend(cache, q, got, lens, tq, window, 0)
        outs.append(cache.attend(0, q, window=60))
    # window 60 of sequence 1: positions 694 .. 699 see 635 .. 699 at most; token 691 is in all of them;
    # of sequence 0: 894 .. 899 see 835 .. 899, token 897 from the fourth query on
    for o in outs[1:]:
        assert torch.equal(o[0, :3], outs[0][0, :3]) and not torch.equal(o[0, 3:], outs[0][0, 3:])


@pytest.mark.gpu
def test_masked_tokens_may_hold_anything(status):
    """NaN and infinities behind the window, behind the sequence and in another sequence change nothing."""
    lens, tq = [200, 90], [1, 1]
    cache = fill(2, 256, 1, 64, lens, tq, torch.float16)
    q = randn(2, 1, 2, 64, seed=55, dtype=torch.float16)
    want = cache.attend(0, q, window=40, sinks=3)
    bad = torch.full((2, 120, 1, 64), float("nan"), device="cuda", dtype=torch.float16)
    bad[:, ::2] = float("inf")
    held = cache.lengths.clone()
    cache.lengths.copy_(torch.tensor([10, 100], dtype=torch.int32))
    cache.append(0, bad, -bad, counts=torch.tensor([120, 60], dtype=torch.int32, device="cuda"))
    cache.lengths.copy_(held)
    assert torch.equal(cache.attend(0, q, window=40, sinks=3), want)


@pytest.mark.gpu
def test_tokens_past_the_end_are_left_out_and_reported(status):
    cache = QuantizedKVCache(1, 2, 1, 64, 40)
    cache.append(0, randn(2, 40, 1, 64), randn(2, 40, 1, 64, seed=1))
    before = cache.pages.clone()
    cache.advance(torch.tensor([40, 39], dtype=torch.int32, device="cuda"))
    k = randn(2, 2, 1, 64, seed=2)
    cache.append(0, k, k)
    st = status()
    assert st["code"] == 5 and st["count"] >= 1  # bounds
    got = cache.read(0, 39, 1, dtype=torch.float32)[0]
    assert torch.equal(got[1, 0], quantize_groups(k[1, 0]).float())
    assert torch.equal(cache.pages[:, 0], before[:, 0])
    o = cache.attend(0, randn(2, 2, 1, 64, seed=3))
    assert status()["code"] == 5 and o.isfinite().all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(status):
    """A layer of 4.6 GB: the last head's last pages."""
    n = 450_000
    cache = QuantizedKVCache(1, 1, 64, 128, n)
    assert cache.nbytes > 1 << 32
    cache.advance(n - 70)
    k, v = randn(1, 70, 64, 128, seed=1), randn(1, 70, 64, 128, seed=2)
    cache.append(0, k, v)
    for got, x in zip(cache.read(0, n - 70, 70, dtype=torch.float32), (k, v)):
        assert torch.equal(got, quantize_groups(x).float())
    cache.advance(69)
    q = randn(1, 1, 64, 128, seed=3)
    got = cache.attend(0, q, window=70)
    kk, vv = (t.double()[0] for t in cache.read(0, n - 70, 70, dtype=torch.float32))
    want, _, _ = attention(q[0].double(), kk, vv, torch.tensor([69], device="cuda"), None, 0, 128**-0.5)
    assert (got[0].double() - want).abs().max() < 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n", [(torch.float32, 131_070 + 3), (torch.bfloat16, 262_140 + 5)])
def test_more_tokens_than_one_grid(dtype, n, status):
    """Appends and reads of more runs of tokens than a grid has in one dimension."""
    cache = QuantizedKVCache(1, 1, 16, 128, n + 1)
    x = randn(1, 1009, 16, 128, seed=1, dtype=dtype)
    k = torch.cat([x] * (n // 1009 + 1), 1)[:, :n]
    cache.append(0, k, -k, counts=torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    want = quantize_groups(x), quantize_groups(-x)
    for got, w in zip(cache.read(0, dtype=torch.float16), want):
        assert got.shape[1] == n + 1
        for at in (0, 130 * 1009, n // 1009 * 1009):
            part = got[:, at : min(at + 1009, n - 1)]
            assert torch.equal(part, w[:, : part.shape[1]].half())
        assert (got[:, n - 1 :] == 0).all()
    cache.advance(n - 1)
    cache.append(0, x[:, :2], x[:, 1:3])
    for got, w in zip(cache.read(0, n - 1, 2, dtype=torch.float32), (x[:, :2], x[:, 1:3])):
        assert torch.equal(got, quantize_groups(w).float())


@pytest.mark.gpu
def test_more_sequences_than_one_grid(status):
    B = 65_535 + 9
    cache = QuantizedKVCache(1, B, 1, 64, 3)
    k, v = randn(B, 2, 1, 64, seed=1), randn(B, 2, 1, 64, seed=2)
    cache.append(0, k, v, counts=2 - torch.arange(B, device="cuda") % 2)
    for got, x in zip(cache.read(0, 0, 2, dtype=torch.bfloat16), (k, v)):
        want = quantize_groups(x).bfloat16()
        want[1::2, 1] = 0
        assert torch.equal(got, want)
    # one visible token: its own value, but for the roundings of s (code - 8) and lo + 8 s and the result's
    got, want = cache.attend(0, k[:, :1]).double(), cache.read(0, 0, 1, dtype=torch.float32)[1].double()
    top = want.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)  # 8 s + |lo + 8 s| <= 3 of the largest
    err = (3 * H16 * top).expand(B, 1, 1, 2, 32).flatten(-2) + 2.0**-8 * want.abs() + 1e-6
    assert ((got - want).abs() <= 1.01 * err).all()


@pytest.mark.gpu
def test_captured_decoding_and_two_streams(status):
    """A captured step (append, attend, advance) replays with the lengths it finds on the device;
    two caches on two streams do not disturb each other."""
    B, H, D, steps = 2, 2, 64, 70

    def tokens(i):
        return [randn(B, 1, H, D, seed=1000 + 3 * i + j) for j in range(3)]

    eager = QuantizedKVCache(1, B, H, D, 96)
    want = []
    for i in range(steps):
        q, k, v = tokens(i)
        eager.append(0, k, v)
        want.append(eager.attend(0, q, window=50, sinks=2))
        eager.advance(1)

    cache = QuantizedKVCache(1, B, H, D, 96)
    q, k, v = tokens(0)

    def step():
        cache.append(0, k, v)
        o = cache.attend(0, q, window=50, sinks=2)
        cache.advance(1)
        return o

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    cache.reset()
    other = QuantizedKVCache(1, B, H, D, 96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(steps):
        for dst, src in zip((q, k, v), tokens(i)):
            dst.copy_(src)
        with torch.cuda.stream(side):
            a, b, c = tokens(i)
            other.append(0, b, c)
            p = other.attend(0, a, window=50, sinks=2)
            other.advance(1)
        graph.replay()
        assert torch.equal(o, want[i]), i
    side.synchronize()
    assert torch.equal(p, want[-1])
    assert cache.lengths.tolist() == [steps] * B


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        QuantizedKVCache(1, 1, 1, 96, 8)
    c = QuantizedKVCache(1, 1, 1, 64, 8)
    x = torch.zeros(1, 1, 1, 64, device="cuda")
    with pytest.raises(TypeError, match="bf16 or fp16"):
        c.attend(0, x)
    with pytest.raises(RuntimeError, match="the cache on"):
        c.append(0, x.cpu(), x.cpu())
    with pytest.raises(RuntimeError, match="counts are on"):
        c.append(0, x, x, counts=torch.ones(1, dtype=torch.int32))
    with pytest.raises(TypeError, match="unsupported dtype"):
        c.append(0, x.double(), x.double())
    with pytest.raises(TypeError, match="reads as"):
        c.read(0, dtype=torch.float64)
    assert c.attend(0, torch.zeros(1, 0, 1, 64, device="cuda", dtype=torch.bfloat16)).shape == (1, 0, 1, 64)
