"""Next-token sampling: CPU path, CUDA kernel and TransformerLM.generate."""

import math

import pytest
import torch

from underhfs import functional as F

INF = math.inf


def reference(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row in Python floats, token by token."""
    order = sorted((i for i in range(len(x)) if x[i] > -INF), key=lambda i: (-x[i], i))
    if not order:
        return -1
    if t <= 0:
        return order[0]
    w = {i: 1.0 if x[i] == x[order[0]] else math.exp((x[i] - x[order[0]]) / t) for i in order}
    if k > 0:
        order = order[:k]
    if p < 1.0:
        total, run, kept = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and run >= p * total:
                break
            kept.append(i)
            run += w[i]
        order = kept
    order = sorted(i for i in order if w[i] >= min(m, 1.0))
    goal, run, last = u * math.fsum(w[i] for i in order), 0.0, -1
    for i in order:
        if w[i] == 0.0:
            continue
        run, last = run + w[i], i
        if run > goal:
            return i
    return last


def rows(n, vocab, seed, dtype=torch.float32, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(n, vocab, generator=g)).to(dtype), torch.rand(n, generator=g)


def check(x, u, device, t=1.0, k=0, p=1.0, m=0.0):
    got = F.sample(x.to(device), u.to(device), temperature=t, top_k=k, top_p=p, min_p=m).torch()
    assert got.dtype == torch.int64 and got.device.type == device
    pick = lambda v, i: float(v[i]) if isinstance(v, torch.Tensor) else v  # noqa: E731
    want = [reference([float(v) for v in x[i]], float(u[i]), pick(t, i), int(pick(k, i)), pick(p, i), pick(m, i))
            for i in range(x.shape[0])]
    assert got.tolist() == want


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7), dict(k=1), dict(k=5), dict(k=10**9), dict(p=0.9), dict(p=0.3),
            dict(p=1e-9), dict(m=0.1), dict(m=1.0), dict(t=1.7, k=40, p=0.8, m=0.02), dict(t=1e-4), dict(t=50.0, p=0.99)]


def special_rows():
    """Rows where a sampler can go wrong: ties, nothing visible, infinities, the type's lowest value."""
    low = torch.finfo(torch.float32).min
    return torch.tensor([
        [0.0] * 9,
        [-INF] * 9,
        [-INF, -INF, 3.0, -INF, -INF, -INF, -INF, -INF, -INF],
        [low] * 9,
        [low, 1.0, low, 1.0, low, 0.5, low, 0.5, low],
        [1.0, INF, 1.0, INF, 0.0, 0.0, 0.0, 0.0, 0.0],
        [-0.0, 0.0, -0.0, 0.0, -1.0, -1.0, -1.0, -1.0, -1.0],
        [-1000.0, -1001.0, -1000.0, -1002.0, -1e30, -1000.5, -3e38, -1000.0, -1001.0],
        [80.0, -80.0, 79.0, 79.0, 79.0, -INF, 78.0, 79.0, 10.0],
    ])


def run_special(device, **kw):
    x = special_rows()
    for u in (0.0, 0.2, 0.5, 0.75, 0.9999999):
        check(x, torch.full((x.shape[0],), u), device, **kw)


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("kw", SETTINGS)
def test_cpu(kw):
    x, u = rows(12, 57, 1)
    check(x, u, "cpu", **kw)
    check((x * 2).round() / 2, u, "cpu", **kw)  # many ties
    run_special("cpu", **kw)


def test_cpu_per_row_and_shapes():
    x, u = rows(6, 31, 2)
    kw = dict(t=torch.tensor([0.0, 0.5, 1.0, 1.0, 2.0, 0.9]), k=torch.tensor([0, 3, 0, 7, -1, 50], dtype=torch.int32),
              p=torch.tensor([1.0, 0.9, 0.5, 1.0, 0.2, 2.0]), m=torch.tensor([0.0, 0.0, 0.2, 0.0, 0.5, 0.01]))
    check(x, u, "cpu", **kw)
    got = F.sample(x.view(2, 3, 31), u.view(2, 3), top_k=4).torch()
    assert torch.equal(got.reshape(-1), F.sample(x, u, top_k=4).torch())
    assert F.sample(x[0], u[0]).torch().shape == ()


def test_nan_is_never_chosen():
    x = torch.tensor([[float("nan"), 1.0, float("nan"), 2.0], [float("nan")] * 4])
    for u in (0.0, 0.5, 0.999):
        got = F.sample(x, torch.full((2,), u), temperature=5.0).torch()
        assert got[0].item() in (1, 3) and got[1].item() == -1


def test_distribution_follows_the_softmax():
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0]])
    n = 4000
    u = (torch.arange(n) + 0.5) / n  # evenly spread: each count is within one of n * probability
    got = F.sample(x.expand(n, 4), u).torch().bincount(minlength=4)
    assert (got - n * torch.softmax(x[0].double(), 0)).abs().max() <= 1


def kernel_weight(l, mx, temperature, exact):
    """The CUDA kernel's integer weight, its fp32 steps one by one (csrc/kernels/sample.cu)."""
    import numpy as np

    f, d64 = np.float32, np.float64
    fma = lambda a, b, c: f(d64(a) * d64(b) + d64(c))  # noqa: E731  (the sum's rounding to 53 bits is far below fp32's)
    c = 1.4426950408889634 / temperature
    ch = f(c)
    cl = f(c - d64(ch))
    l, mx = f(l), f(mx)
    d0, dmin = l - mx, f(f(-44.9) / ch)
    d = np.maximum(d0, dmin)
    p = d * ch
    q = fma(d, cl, fma(d, ch, -p))
    if exact:
        bb = d0 - l
        e = (l - (d0 - bb)) + (-mx - bb)
        q = fma(np.where(d0 < dmin, f(0), e), ch, q)
    z = np.rint(d64(p) * 64)  # the sum with 1.5 * 2^23 rounds to a whole number
    r = fma(f(z), f(-1 / 64), p) + q
    em1 = r * fma(r, fma(r, f(0.055504109), f(0.24022651)), f(0.69314718))
    k = z.astype(np.int64)
    m0 = np.floor(2.0 ** ((k & 63) / 64.0) * 2.0**30 + 0.5).astype(np.int64)
    m = m0 + np.rint(m0.astype(f) * em1).astype(np.int64)
    return (m << 14) >> -(k >> 6)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 1.3, 30.0])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "near", "wide"])
def test_kernel_weights_hold_their_error(temperature, kind):
    """2^-29 of the weight and one unit of 2^-44: r, the series, its product with the table's
    entry and the conversion round to 2^-24 of at most 2^-7.5, about six times; the table to 2^-31."""
    import numpy as np

    g = np.random.default_rng(1)
    mx = np.float32({"fp32": 11.7, "bf16": 13.0625, "near": 7.1, "wide": 900.0}[kind])
    l = (mx - np.abs(g.standard_normal(200000)) * 8 * temperature).astype(np.float32)
    if kind == "bf16":
        l = torch.from_numpy(l).bfloat16().float().numpy()
    if kind == "near":
        l = (mx - np.abs(g.standard_normal(200000)) * 1e-3).astype(np.float32)
    l = np.minimum(l, mx)
    want = np.exp((l.astype(np.float64) - np.float64(mx)) / temperature) * 2.0**44
    for exact in (True, False) if kind == "bf16" else (True,):  # without the difference's error: 16-bit logits
        got = kernel_weight(l, mx, temperature, exact).astype(np.float64)
        near = np.abs(l) > np.abs(mx) * 2.0**-14 if not exact else np.full(l.shape, True)
        assert (np.abs(got - want) <= want * 2.0**-29 + 1)[near].all()
        assert kernel_weight(np.full(3, mx), mx, temperature, exact).tolist() == [2**44] * 3
        far = np.array([-3.4e38, -np.inf, mx - 50 * temperature], dtype=np.float32)
        assert kernel_weight(far, mx, temperature, exact).tolist() == [0, 0, 0]


def test_rounded_weights_of_a_run_sum_to_its_sum():
    """The kernel's rounding of weights to 2^-31 for top-p's border (coarse() in csrc/kernels/sample.cu): over any run of
    tokens the sum is off by some units, whatever the weight.  (The thresholds are multiples of the golden ratio
    modulo 1: of n of them, n x lie below x but for a few times log n.)"""
    import numpy as np

    idx = np.arange(327680, dtype=np.int64)
    t = ((idx * 0x9E3779B1) & 0xFFFFFFFF) >> 19
    assert t.max() == 2**13 - 1 and ((2**44 + t) >> 13).max() == 2**31  # the largest stays the largest
    g = np.random.default_rng(0)
    for w in [1, 2, 3629, 4095, 4096, 4097, 8191, 8192, 12345, *g.integers(1, 1 << 16, 20)]:
        run = np.concatenate(([0], np.cumsum((int(w) + t) >> 13)))
        off = run - np.arange(len(run)) * (w / 8192)
        assert off.max() - off.min() <= 32  # of any run: off at its end minus off at its start


@pytest.mark.parametrize("kw,match", [
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(top_k=-1), "top_k"), (dict(top_p=1.5), "top_p"), (dict(top_p=-0.1), "top_p"),
    (dict(min_p=float("nan")), "min_p"), (dict(min_p=1.1), "min_p"),
    (dict(temperature=torch.ones(3)), "temperature needs one value"),
])
def test_refuses_settings(kw, match):
    with pytest.raises(ValueError, match=match):
        F.sample(torch.zeros(2, 5), torch.zeros(2), **kw)


def test_large_top_k_is_off():
    """int64 values beyond 32 bits do not wrap round to small ones."""
    x, u = torch.randn(3, 40), torch.rand(3)
    k = torch.tensor([2**32 + 1, 2**31 + 7, -(2**32) + 2])
    assert torch.equal(F.sample(x, u, top_k=k).torch(), F.sample(x, u).torch())


def test_refuses_shapes_and_types():
    with pytest.raises(ValueError, match="uniform"):
        F.sample(torch.zeros(2, 5), torch.zeros(3))
    with pytest.raises(ValueError, match="vocab"):
        F.sample(torch.zeros(2, 0), torch.zeros(2))
    with pytest.raises(TypeError, match="floating"):
        F.sample(torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2))


# ------------------------------------------------------------------- GPU
@pytest.fixture
def status_ok():
    yield
    from underhfs_b200.ops._lib import core

    st = core().device_status(True)
    assert st["code"] == 0, st


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS)
def test_gpu_special_rows(kw, status_ok):
    run_special("cuda", **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 2), (5, 63), (2, 1001), (1, 5000), (300, 129), (2, 33001)])
def test_gpu_sizes(n, vocab, dtype, status_ok):
    x, u = rows(n, vocab, n + vocab, dtype)
    for kw in (dict(), dict(t=0.8, p=0.9), dict(k=50, p=0.95, m=0.01), dict(t=0.0), dict(k=max(1, vocab // 2))):
        check(x, u, "cuda", **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [4096, 40000])
@pytest.mark.parametrize("kw", [dict(k=1500), dict(k=3000, p=0.7), dict(p=0.9), dict(p=0.999, m=0.5), dict(t=0.3, p=0.2)])
def test_gpu_long_runs_of_equal_logits(vocab, kw, status_ok):
    """More tokens at the border than the kernel compares at once: the key's bits decide, then the index."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-1, 2, (2, vocab), generator=g).float()
    x = torch.cat((x, torch.full((1, vocab), 2.5), torch.arange(vocab).float().unsqueeze(0) * 1e-6 + 7.0))
    for u in (0.0, 0.31, 0.999):
        check(x, torch.full((4,), u), "cuda", **kw)
    check(x.bfloat16(), torch.full((4,), 0.6), "cuda", **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("kw", [dict(k=200, p=0.8), dict(p=0.95), dict(p=0.99999), dict(t=20.0, p=0.9), dict(k=257),
                                dict(t=0.0), dict(m=0.2)])
def test_gpu_largest_vocabulary(kw, dtype, status_ok):
    x, u = rows(2, 327680, 31, dtype)
    check(x, u, "cuda", **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(p=0.9), dict(k=100, p=0.95), dict(k=100), dict(k=1000, p=0.6)])
@pytest.mark.parametrize("shift", [0.0, 900.0, -30000.0])
def test_gpu_list_and_slices_agree(kw, shift, status_ok):
    """Peaked rows (a short list does) and flat ones (it does not), near 0 and far from it."""
    for scale, t in ((4.0, 0.5), (0.01, 1.0), (3.0, 1e-4), (3.0, 60.0)):
        x, u = rows(3, 9001, 41, scale=scale)
        check(x + shift, u, "cuda", t=t, **kw)


@pytest.mark.gpu
def test_gpu_per_row_settings_strides_and_alignment(status_ok):
    big, u = rows(8, 4100, 9)
    kw = dict(t=torch.tensor([0.0, 0.5, 1.0, 1.0, 2.0, 0.9, 1.1, 0.7]),
              k=torch.tensor([0, 3, 0, 700, -1, 5000, 1, 9], dtype=torch.int32),
              p=torch.tensor([1.0, 0.9, 0.5, 1.0, 0.2, 2.0, 0.9, 0.0]),
              m=torch.tensor([0.0, 0.0, 0.2, 0.0, 0.5, 0.01, 0.3, 0.0]))
    dev = {n: v.cuda() for n, v in kw.items()}
    x = big.cuda()
    for view in (x, x[:, 1:], x[:, 3:2050], x.t().contiguous().t()):
        cpu = view.cpu()
        got = F.sample(view, u.cuda(), temperature=dev["t"], top_k=dev["k"], top_p=dev["p"], min_p=dev["m"]).torch()
        want = [reference(cpu[i].tolist(), float(u[i]), float(kw["t"][i]), int(kw["k"][i]), float(kw["p"][i]),
                          float(kw["m"][i])) for i in range(8)]
        assert got.tolist() == want


@pytest.mark.gpu
def test_gpu_nan_and_odd_uniforms(status_ok):
    x = torch.tensor([[float("nan"), 1.0, float("nan"), 2.0], [float("nan")] * 4, [0.0, 1.0, 2.0, -INF],
                      [0.0, 1.0, 2.0, -INF], [0.0, 1.0, 2.0, -INF]], device="cuda")
    u = torch.tensor([0.0, 0.5, 1.0, -3.0, float("nan")], device="cuda")
    assert F.sample(x, u).torch().tolist() == [1, -1, 2, 0, 0]


@pytest.mark.gpu
def test_gpu_same_choice_however_the_row_is_split(status_ok):
    """One row takes a cluster of blocks, 400 equal rows one block each."""
    x, _ = rows(1, 30000, 11)
    u = torch.rand(400, generator=torch.Generator().manual_seed(3))
    many = F.sample(x.cuda().expand(400, -1).contiguous(), u.cuda(), temperature=1.3, top_p=0.97).torch()
    one = [F.sample(x.cuda(), u[i : i + 1].cuda(), temperature=1.3, top_p=0.97).torch().item() for i in range(0, 400, 7)]
    assert many.cpu()[::7].tolist() == one


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(t=0.0), dict(k=30, p=0.9), dict(k=5000), dict(p=0.95, m=0.01), dict(t=30.0, p=0.999)])
@pytest.mark.parametrize("n,vocab,dtype", [(230, 20001, torch.float32), (224, 17000, torch.float32),
                                           (60, 70002, torch.float32), (64, 70000, torch.float32),
                                           (240, 40001, torch.bfloat16)])
def test_gpu_many_wide_rows(n, vocab, dtype, kw, status_ok):
    """Rows that the kernel reads again instead of keeping them: the reference's choice, and that of
    each row by itself, with infinities, NaN, long runs and rows of one kind among them."""
    x, u = rows(n, vocab, vocab, dtype)
    x[1] = -INF
    x[2, 5:] = -INF
    x[3] = 0.5
    x[4, ::3] = float("nan")
    x[5] = float("nan")
    x[6, 7::1000] = INF
    x[7] = (x[7] * 2).round() / 2
    x[8, : vocab // 2] = torch.finfo(dtype).min
    got = F.sample(x.cuda(), u.cuda(), temperature=kw.get("t", 1.0), top_k=kw.get("k", 0), top_p=kw.get("p", 1.0),
                   min_p=kw.get("m", 0.0)).torch().tolist()
    for i in [*range(9), n // 2, n - 1]:
        row = [float(v) if v == v else -INF for v in x[i]]
        assert got[i] == reference(row, float(u[i]), **kw), i
    for i in range(0, n, 3):
        assert got[i] == F.sample(x[i : i + 1].cuda(), u[i : i + 1].cuda(), temperature=kw.get("t", 1.0),
                                  top_k=kw.get("k", 0), top_p=kw.get("p", 1.0), min_p=kw.get("m", 0.0)).torch().item(), i


@pytest.mark.gpu
def test_gpu_captured_and_replayed_and_other_stream(status_ok):
    x, u = rows(4, 9000, 21)
    xd, ud = x.cuda(), u.cuda()
    F.sample(xd, ud, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.sample(xd, ud, top_p=0.9).torch()
    for seed in (22, 23):
        y, w = rows(4, 9000, seed)
        xd.copy_(y)
        ud.copy_(w)
        graph.replay()
        want = [reference(y[i].tolist(), float(w[i]), p=0.9) for i in range(4)]
        assert out.tolist() == want
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.sample(xd, ud, top_p=0.9).torch()
    side.synchronize()
    assert got.tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab", [(1, 131072), (70, 131072), (3, 40001), (300, 50000)])
@pytest.mark.parametrize("tail,p", [(-22.3, 0.99999), (-21.0, 0.9999), (-21.0, 0.99995), (-20.6, 0.99992), (-23.75, 0.999999)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_top_p_over_a_long_flat_tail(n, vocab, tail, p, dtype, status_ok):
    """One likely token and a long tail whose weights are near the unit of top-p's histogram: the tokens kept are
    those of exact arithmetic but for 64 units of 2^-31 of the largest weight (a run's rounding, at
    the two ends of what is summed), 2^-29 of the tail and 2^-44 a token."""
    x = torch.full((n, vocab), tail).to(dtype)
    x[:, 0] = 0
    w = math.exp(float(x[0, 1]))
    last = F.sample(x.cuda(), torch.ones(n, device="cuda"), top_p=p).torch()  # u = 1: the last token kept
    goal, off = p * (1 + (vocab - 1) * w), 64 * 2.0**-31 + (vocab - 1) * (w * 2.0**-29 + 2.0**-44)
    fewest, most = (max(0, math.ceil((g - 1) / w)) for g in (goal - off, goal + off))
    assert fewest <= last.min().item() and last.max().item() <= most, (fewest, last, most)
    assert (last == last[0]).all()


@pytest.mark.gpu
def test_gpu_refusals():
    with pytest.raises(ValueError, match="vocabularies up to"):
        F.sample(torch.zeros(1, 327681, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(RuntimeError, match="uniform is on"):
        F.sample(torch.zeros(1, 40, device="cuda"), torch.zeros(1))
    with pytest.raises(RuntimeError, match="top_p is on"):
        F.sample(torch.zeros(1, 40, device="cuda"), torch.zeros(1, device="cuda"), top_p=torch.ones(1))
    assert F.sample(torch.zeros(0, 40, device="cuda"), torch.zeros(0, device="cuda")).torch().shape == (0,)
