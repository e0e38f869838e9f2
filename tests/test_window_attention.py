"""Causal attention with a sliding window and sinks: CPU layers, the tcgen05 kernels, refusals."""

import math

import pytest
import torch

from underhfs.nn import CausalSelfAttention, SelfAttention, TransformerLM
from underhfs.tensor import Tensor
from underhfs_b200.models.transformer import LMSpec
from underhfs_b200.ops.kernels import window_args

HALF = torch.finfo(torch.bfloat16).eps / 2  # one rounding to bf16, relative


def visible(T, window, sinks, device="cpu"):
    i = torch.arange(T, device=device)[:, None]
    j = torch.arange(T, device=device)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def oracle(qkv, do, B, T, H, D, window, sinks):
    """(o, dqkv) in 64 bits and, element by element, the most that the kernels'
    bf16 roundings can move them.

    The forward rounds each probability (P) and the output; the backward
    rounds P, dS and the gradients, and takes delta = sum(dO * O) from the
    rounded O.  A rounding is off by at most HALF of its value.
    """
    x = qkv.double().view(B, T, 3, H, D).permute(2, 0, 3, 1, 4)
    q, k, v = x[0], x[1], x[2]
    scale = 1.0 / math.sqrt(D)
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~visible(T, window, sinks, qkv.device), float("-inf"))
    p = torch.softmax(s, -1)
    o = p @ v
    o_err = HALF * (p @ v.abs() + o.abs())
    g = do.double().view(B, T, H, D).permute(0, 2, 1, 3)
    dv = p.transpose(-1, -2) @ g
    dv_err = HALF * (p.transpose(-1, -2) @ g.abs() + dv.abs())
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (g @ v.transpose(-1, -2) - delta)
    ds_err = HALF * ds.abs() + p * (g.abs() * o_err).sum(-1, keepdim=True)
    dq, dk = scale * ds @ k, scale * ds.transpose(-1, -2) @ q
    dq_err = scale * ds_err @ k.abs() + HALF * dq.abs()
    dk_err = scale * ds_err.transpose(-1, -2) @ q.abs() + HALF * dk.abs()
    grad = torch.stack((dq, dk, dv)).permute(1, 3, 0, 2, 4).reshape(B * T, 3 * H * D)
    grad_err = torch.stack((dq_err, dk_err, dv_err)).permute(1, 3, 0, 2, 4).reshape(B * T, 3 * H * D)
    flat = lambda t: t.permute(0, 2, 1, 3).reshape(B * T, H * D)  # noqa: E731
    return flat(o), flat(o_err), grad, grad_err


def within(got, want, err):
    # fp32 sums, ex2 and the log-sum-exp add about 2^-17 of each term
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - (1.01 * err + 1e-6)
    assert over.max().item() <= 0, f"beyond its roundings by {over.max().item():.3g}"


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (5, 40), (64, 1)])
def test_cpu_layer_matches_the_formula(window, sinks):
    torch.manual_seed(0)
    layer = CausalSelfAttention(8, heads=2, window=window, sinks=sinks)
    for p in layer.parameters():
        p._data.data.copy_(torch.randn_like(p._data))
    x = torch.randn(2, 9, 8, dtype=torch.float64)
    got = layer(Tensor._wrap(x))._data

    def lin(m, t):
        return t @ m.weight._data.t() + m.bias._data

    q, k, v = (lin(m, x).view(2, 9, 2, 4).transpose(1, 2) for m in (layer.q_proj, layer.k_proj, layer.v_proj))
    s = (q @ k.transpose(-1, -2)) / 2.0
    s = s.masked_fill(~visible(9, window, sinks), float("-inf"))
    want = lin(layer.out_proj, (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(2, 9, 8))
    assert torch.allclose(got, want, rtol=0, atol=1e-12)


def test_cpu_wide_window_is_plain_attention():
    kw = dict(vocab_size=32, max_seq_len=12, features=8, hidden_features=16, layers=2, heads=2)
    ids = torch.arange(12) % 7
    a = TransformerLM(**kw)(ids)._data
    b = TransformerLM(**kw, window=12, sinks=3)(ids)._data
    c = TransformerLM(**kw, window=3)(ids)._data
    assert torch.equal(a, b)
    assert torch.equal(a[:3], c[:3]) and not torch.equal(a[3:], c[3:])


def test_window_arguments():
    assert window_args(100, True, None, 0) == (0, 0)
    assert window_args(100, True, 100, 7) == (0, 0)
    assert window_args(100, True, 99, 700) == (99, 100)
    for bad in ((None, 3), (0, 0), (-4, 0), (5, -1)):
        with pytest.raises(ValueError):
            window_args(100, True, *bad)
    with pytest.raises(ValueError, match="causal"):
        window_args(100, False, 5, 0)
    with pytest.raises(ValueError, match="causal"):
        SelfAttention(8, window=4)
    with pytest.raises(ValueError, match="window"):
        TransformerLM(32, 8, 8, 8, 1, window=0)
    with pytest.raises(ValueError, match="sinks"):
        TransformerLM(32, 8, 8, 8, 1, sinks=2)


def test_flops_count_the_visible_keys():
    def spec(**kw):
        return LMSpec(1000, 512, 64, 256, 2, heads=1, **kw)

    T, w, s = 512, 100, 9
    full = spec().train_flops_per_token(T)
    part = spec(window=w, sinks=s).train_flops_per_token(T)
    pairs = visible(T, w, s).sum().item()
    per_pair = 2 * 3 * 2 * 2 * 64 / T
    # the count takes an integral for a sum: off by at most one key a token on either side
    assert abs((full - part) - per_pair * (T * (T + 1) / 2 - pairs)) <= 2 * per_pair * T
    assert spec(window=T).train_flops_per_token(T) == full


# ------------------------------------------------------------------- GPU
CASES = [  # B, T, H, D, window, sinks
    (1, 2, 1, 64, 1, 0),
    (2, 130, 2, 64, 33, 1),
    (2, 300, 2, 64, 1, 0),
    (1, 300, 1, 128, 1, 2),
    (1, 257, 1, 128, 128, 0),
    (2, 400, 1, 64, 399, 0),
    (1, 385, 1, 64, 127, 128),
    (1, 640, 1, 64, 129, 130),
    (1, 777, 1, 128, 64, 700),
    (1, 1024, 2, 64, 256, 4),
    (1, 1100, 1, 128, 300, 257),
    (3, 513, 3, 64, 200, 5),
]


def _inputs(B, T, H, D, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(B * T, 3 * H * D, generator=g, device="cuda").to(torch.bfloat16)
    do = torch.randn(B * T, H * D, generator=g, device="cuda").to(torch.bfloat16)
    return qkv, do


def _run(qkv, do, B, T, H, D, window, sinks):
    from underhfs_b200.ops.functions import flash_attention

    x = qkv.detach().requires_grad_(True)
    o = flash_attention(x, B, T, H, D, True, window=window, sinks=sinks)
    return o.detach(), torch.autograd.grad(o, x, do)[0]


@pytest.fixture
def status_ok():
    yield
    from underhfs_b200.ops._lib import core

    st = core().device_status(True)
    assert st["code"] == 0, st


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,D,window,sinks", CASES)
def test_forward_backward(B, T, H, D, window, sinks, status_ok):
    qkv, do = _inputs(B, T, H, D)
    o, dqkv = _run(qkv, do, B, T, H, D, window, sinks)
    want, err, grad, grad_err = oracle(qkv, do, B, T, H, D, window, sinks)
    within(o, want, err)
    within(dqkv, grad, grad_err)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [200, 5000])
def test_wide_window_is_the_plain_kernel(window, status_ok):
    qkv, do = _inputs(2, 200, 2, 64)
    a = _run(qkv, do, 2, 200, 2, 64, None, 0)
    b = _run(qkv, do, 2, 200, 2, 64, window, 3)
    assert torch.equal(a[0], b[0])
    # dQ is summed with atomic adds: equal but for the order of the sum
    assert torch.allclose(a[1].float(), b[1].float(), rtol=2 * HALF, atol=1e-3)


@pytest.mark.gpu
def test_gradient_against_differences(status_ok):
    B, T, H, D, window, sinks = 1, 300, 1, 64, 100, 3
    qkv, do = _inputs(B, T, H, D, 3)
    _, dqkv = _run(qkv, do, B, T, H, D, window, sinks)
    _, _, _, err = oracle(qkv, do, B, T, H, D, window, sinks)
    g = torch.Generator(device="cuda").manual_seed(4)
    way = torch.randn(qkv.shape, generator=g, device="cuda", dtype=torch.float64)

    def f(x):
        return (oracle(x, do, B, T, H, D, window, sinks)[0] * do.double()).sum()

    h = 1e-4
    want = (f(qkv.double() + h * way) - f(qkv.double() - h * way)) / (2 * h)
    got = (dqkv.double() * way).sum()
    # the gradient's own error bound along the direction; the difference quotient's h^2 term is far below it
    assert (got - want).abs() <= (err * way.abs()).sum()


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,D,window,sinks", [(16, 1024, 12, 64, 256, 4), (2, 2048, 16, 128, 500, 4)])
def test_many_blocks_per_processor(status_ok, B, T, H, D, window, sinks):
    """Each multiprocessor walks many key blocks: dK and dV, summed in a fixed order, come out
    in the same bits every time; dQ, summed by atomics, within a bf16 rounding; and all of
    a head agrees with 64 bits."""
    qkv, do = _inputs(B, T, H, D)
    first = _run(qkv, do, B, T, H, D, window, sinks)
    F = H * D
    for _ in range(12):
        o, grad = _run(qkv, do, B, T, H, D, window, sinks)
        assert torch.equal(o, first[0])
        assert torch.equal(grad[:, F:], first[1][:, F:])
        # fp32 sums of at most 17 tiles in another order, then a rounding each: a step apart
        off = (grad[:, :F].double() - first[1][:, :F].double()).abs()
        assert (off <= 2.02 * HALF * first[1][:, :F].double().abs() + 1e-5).all()
    heads = torch.arange(0, H, 5, device="cuda")
    part = lambda t, n: t.view(B, T, n, H, D)[:, :, :, heads].reshape(B * T, -1)  # noqa: E731
    o, o_err, want, err = oracle(part(qkv, 3), part(do, 1), B, T, len(heads), D, window, sinks)
    within(part(first[0], 1), o, o_err)
    within(part(first[1], 3), want, err)


@pytest.mark.gpu
def test_sequences_do_not_touch_each_other(status_ok):
    """A ragged last block reads zeros, not the next sequence (here infinities and NaN)."""
    B, T, H, D = 3, 130, 1, 64
    qkv, do = _inputs(B, T, H, D)
    want = _run(qkv, do, B, T, H, D, 40, 2)
    qkv[T : 2 * T] = float("nan")
    do[T : 2 * T] = float("inf")
    got = _run(qkv, do, B, T, H, D, 40, 2)
    for a, b in zip(got, want):
        for rows in (slice(0, T), slice(2 * T, 3 * T)):
            assert torch.allclose(a[rows].float(), b[rows].float(), rtol=2 * HALF, atol=1e-3)


@pytest.mark.gpu
def test_captured_and_replayed(status_ok):
    B, T, H, D = 2, 260, 2, 64
    qkv, do = _inputs(B, T, H, D)
    from underhfs_b200.ops import kernels as K

    def step(x, g):
        o, lse = K.flash_attn_qkv(x, B, T, H, D, True, window=50, sinks=4)
        return o, K.flash_attn_qkv_backward(x, o, lse, g, B, T, H, D, True, window=50, sinks=4)

    step(qkv, do)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(qkv, do)
    for seed in (7, 8):
        x, g = _inputs(B, T, H, D, seed)
        qkv.copy_(x)
        do.copy_(g)
        graph.replay()
        want, err, grad, grad_err = oracle(x, g, B, T, H, D, 50, 4)
        within(out[0], want, err)
        within(out[1], grad, grad_err)


def test_forward_mode_is_refused(monkeypatch):
    """There is no forward-mode rule: a dual tensor is refused, not passed on without its tangent."""
    import torch.autograd.forward_ad as fwd

    from underhfs_b200.ops import functions as OF

    def plain(qkv, B, T, H, D, causal, scale=None, window=None, sinks=0):
        q, k, v = qkv.view(B, T, 3, H, D).permute(2, 0, 3, 1, 4)
        s = (q @ k.mT * D**-0.5).masked_fill(torch.ones(T, T).triu(1).bool(), float("-inf"))
        return (s.softmax(-1) @ v).transpose(1, 2).reshape(B * T, H * D), None

    monkeypatch.setattr(OF.K, "flash_attn_qkv", plain)
    x = torch.randn(8, 3 * 64, generator=torch.Generator().manual_seed(0))
    call = lambda t: OF.flash_attention(t, 1, 8, 1, 64, True)  # noqa: E731
    want = call(x)
    assert torch.equal(call(x.clone().requires_grad_(True)).detach(), want)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            call(fwd.make_dual(x, torch.ones_like(x)))
        assert torch.equal(call(x), want)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(x.unsqueeze(0))


def test_refuses_cpu_tensors():
    from underhfs_b200.ops.functions import flash_attention

    with pytest.raises(RuntimeError, match="CUDA"):
        flash_attention(torch.zeros(32, 192, dtype=torch.bfloat16), 1, 32, 1, 64, True, window=4)


@pytest.mark.gpu
def test_refusals():
    from underhfs_b200.ops import kernels as K
    from underhfs_b200.ops.functions import flash_attention

    x = torch.zeros(32, 3 * 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="causal"):
        flash_attention(x, 1, 32, 1, 64, False, window=4)
    with pytest.raises(ValueError, match="bf16"):
        flash_attention(x.half(), 1, 32, 1, 64, True, window=4)
    with pytest.raises(ValueError, match="qkv must be"):
        flash_attention(x, 1, 64, 1, 64, True, window=4)
    odd = torch.zeros(32 * 192 + 8, device="cuda", dtype=torch.bfloat16)[1 : 1 + 32 * 192].view(32, 192)
    with pytest.raises(RuntimeError, match="16-byte"):
        K.flash_attn_qkv(odd, 1, 32, 1, 64, True, window=4)


@pytest.mark.gpu
def test_engine_trains_with_a_window(status_ok):
    """Loss and gradients of a windowed TransformerLM against the same model in 64 bits on the CPU."""
    kw = dict(vocab_size=128, max_seq_len=200, features=128, hidden_features=256, layers=2, heads=2, window=40,
              sinks=3, init="normal", seed=1)
    cpu, gpu = TransformerLM(**kw), TransformerLM(**kw).to("cuda", dtype="bf16")
    for (_, a), (_, b) in zip(cpu.named_parameters(), gpu.named_parameters()):
        a._data.data.copy_(b._data.double().cpu())  # the same bf16 weights
    ids = torch.randint(0, 128, (2, 200))
    tg = torch.randint(0, 128, (2, 200))
    la = cpu(ids, tg)
    la.backward()
    gpu.zero_grad()
    lb = gpu(ids.cuda(), tg.cuda())
    lb.backward()
    # a loss near ln(128) whose logits pass through two blocks of bf16 activations
    assert abs(la.item() - lb.item()) < 8 * HALF * la.item()
    want = {name: p._data.grad for name, p in cpu.named_parameters()}
    for name, p in gpu.named_parameters():
        x, y = want[name], p._main_grad.double().cpu()
        # A key bias shifts all scores of a query alike, so its gradient, the sum of
        # dK over the tokens, is 0 and only dK's roundings are left of it: HALF times
        # the norm of the summands at most.  The weight's gradient sums the same dK
        # times the normalised inputs (root mean square 1) and is of at least that size.
        size = want[name.replace("bias", "weight")] if name.endswith("k_proj.bias") else x
        assert (x - y).norm() <= 16 * HALF * size.norm() + 1e-7, name
