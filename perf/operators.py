"""Timed cases of the long-context and serving operators.

Four operators that belong together when a language model is trained on, or
answers from, long contexts:

* ``window``  causal attention with a sliding window whose first tokens (the
  sinks) stay visible, forward and backward, over a fused q|k|v projection;
* ``write``   keys and values quantised to 4 bits as they enter the cache, and
  read back;
* ``attend``  attention of new tokens over that cache, ragged lengths, shared
  key/value heads, with the same window and sinks;
* ``sample``  the next token from the logits with temperature, top-k, top-p
  and min-p, from given uniform numbers.

With ``own = False`` ``run`` computes each in plain torch operations; with
``own = True`` it calls this package.

The 4-bit format (both sides): channels in groups of 32 of one token and head;
``lo = fp16(min)``, ``s = fp16(fp32(max - lo) / 15)``, code
``round_half_even((x - lo) / s)`` clamped to 0..15 (0 where s is 0), standing
for ``lo + s * code``.
"""

from __future__ import annotations

import math

import torch

own = False

GROUP = 32
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one training step's attention of a 12 x 64 model, 16 sequences of 1024
        dict(name="window-train-16x1024-12x64", op="window", B=16, T=1024, H=12, D=64, window=256, sinks=4,
             train=True),
        # the attention of one layer of a 32 x 128 model trained on 4096 tokens
        dict(name="window-train-2x4096-32x128", op="window", B=2, T=4096, H=32, D=128, window=1024, sinks=4,
             train=True),
        # a long prompt read by an inference program
        dict(name="window-prompt-1x16384-16x128", op="window", B=1, T=16384, H=16, D=128, window=2048, sinks=64,
             train=False),
        # a short prompt of odd length in a model with few heads
        dict(name="window-prompt-1x333-4x64", op="window", B=1, T=333, H=4, D=64, window=100, sinks=3, train=False),
        # the tokens of 32 running sequences entering the cache of one layer
        dict(name="write-token-32x1-32x128", op="write", B=32, T=1, H=32, D=128, dtype="bf16", start=1777,
             ragged=False),
        # a batch of prompts of different lengths entering the cache
        dict(name="write-prompt-8x2048-16x128", op="write", B=8, T=2048, H=16, D=128, dtype="bf16", start=0,
             ragged=True),
        # one interactive sequence of a 12 x 64 model near its longest context
        dict(name="attend-token-1x1000-12x64", op="attend", B=1, Tq=1, keys=1000, Hq=12, Hkv=12, D=64, window=0,
             sinks=0, dtype="bf16"),
        # 32 running sequences of a 32 x 128 model
        dict(name="attend-token-32x4096-32x128", op="attend", B=32, Tq=1, keys=4096, Hq=32, Hkv=32, D=128, window=0,
             sinks=0, dtype="bf16"),
        # a few drafted tokens checked at once over long windowed contexts, 4 query heads to a key/value head
        dict(name="attend-draft-4x30001-32q8x128", op="attend", B=4, Tq=5, keys=30001, Hq=32, Hkv=8, D=128,
             window=8192, sinks=4, dtype="bf16"),
        # one interactive sequence choosing its next token
        dict(name="sample-1x32000", op="sample", rows=1, vocab=32000, dtype="bf16", per_row=False, temperature=0.8,
             top_k=0, top_p=0.95, min_p=0.0, masked=0.0),
        # a serving batch in which every request brings its own settings
        dict(name="sample-256x32000-mixed", op="sample", rows=256, vocab=32000, dtype="bf16", per_row=True,
             temperature=1.0, top_k=50, top_p=0.9, min_p=0.05, masked=0.0),
        # a large vocabulary with a grammar that forbids most of it
        dict(name="sample-64x131072-masked", op="sample", rows=64, vocab=131072, dtype="fp32", per_row=False,
             temperature=1.3, top_k=0, top_p=0.98, min_p=0.0, masked=0.6),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["window", "write", "attend", "sample"])
    D = rng.choice([64, 128])
    if op == "window":
        T = _log_int(rng, 1, 8192)
        window = _log_int(rng, 1, T + 64)
        sinks = rng.choice([0, _log_int(rng, 1, 300)])
        H = _log_int(rng, 1, 32)
        B = _log_int(rng, 1, 16)
        while B * H * D * T * min(T, window + sinks + 256) > 32 * 128 * 4096 * 1280 or B * T * H * D > 1 << 25:
            B, H = max(1, B // 2), max(1, H - H // 3 if H > 1 else 1)
        return dict(op=op, B=B, T=T, H=H, D=D, window=window, sinks=sinks, train=rng.random() < 0.6)
    if op == "write":
        B, T, H = _log_int(rng, 1, 32), _log_int(rng, 1, 4096), _log_int(rng, 1, 32)
        while B * T * H * D > 8 * 2048 * 16 * 128:
            B, T = max(1, B // 2), max(1, T - T // 3)
        return dict(op=op, B=B, T=T, H=H, D=D, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    start=rng.choice([0, _log_int(rng, 1, 3000)]), ragged=rng.random() < 0.5)
    if op == "attend":
        Hkv, ratio = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 3, 4, 8])
        Hkv = max(1, min(Hkv, 64 // ratio))
        Tq = rng.choice([1, 1, _log_int(rng, 2, 24)])
        keys = _log_int(rng, Tq, 32768)
        B = _log_int(rng, 1, 32)
        while B * Hkv * keys * D * max(1.0, Tq * ratio / 16) > 32 * 32 * 4096 * 128:
            B, Hkv = max(1, B // 2), max(1, Hkv // 2)
            keys = max(Tq, keys - keys // 8)
        windowed = rng.random() < 0.4
        return dict(op=op, B=B, Tq=Tq, keys=keys, Hq=Hkv * ratio, Hkv=Hkv, D=D,
                    window=_log_int(rng, 1, keys + 10) if windowed else 0,
                    sinks=rng.choice([0, _log_int(rng, 1, 200)]) if windowed else 0,
                    dtype=rng.choice(["bf16", "fp16"]))
    rows, vocab = _log_int(rng, 1, 256), _log_int(rng, 2, 131072)
    while rows * vocab > 64 * 131072:
        rows = max(1, rows // 2)
    return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                per_row=rng.random() < 0.5, temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.5]),
                top_k=rng.choice([0, _log_int(rng, 1, vocab)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95]),
                min_p=rng.choice([0.0, 0.02, 0.1]), masked=rng.choice([0.0, 0.5]))


# ------------------------------------------------------------------ the inputs
def _lengths(case):
    """Keys of each sequence (its new tokens included): between half of and all of ``keys``."""
    n, tq = case["keys"], case["Tq"]
    return [max(tq, n - (b * 7919) % (n // 2 + 1)) for b in range(case["B"])]


def _counts(case):
    """Tokens that each prompt of a write brings."""
    T = case["T"]
    if not case["ragged"]:
        return [T] * case["B"]
    return [max(1, T - (b * 7919) % (T // 2 + 1)) for b in range(case["B"])]


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _keys_values(B, T, H, D, gen, dtype):
    # keys have channels with a constant offset, as projections with a bias do
    k = torch.randn((B, T, H, D), generator=gen, device="cuda", dtype=torch.float32)
    k += 2.0 * torch.randn((1, 1, H, D), generator=gen, device="cuda", dtype=torch.float32)
    v = torch.randn((B, T, H, D), generator=gen, device="cuda", dtype=torch.float32)
    return k.to(dtype), v.to(dtype)


def _logits(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    # a few likely tokens and a long tail: log-rank slope with noise, the ranks shuffled for each row
    rank = torch.argsort(torch.rand((rows, vocab), generator=gen, device="cuda"), dim=1).float()
    x = 12.0 - 1.4 * torch.log(rank + 1.0)
    x += 0.7 * torch.randn((rows, vocab), generator=gen, device="cuda")
    if case["masked"]:
        drop = torch.rand((rows, vocab), generator=gen, device="cuda") < case["masked"]
        drop[:, 0] = False
        x = x.masked_fill(drop, -math.inf)
    return x.to(_DTYPES[case["dtype"]])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    op = case["op"]
    if op == "window":
        B, T, F = case["B"], case["T"], case["H"] * case["D"]
        x = {"qkv": _randn((B * T, 3 * F), gen, torch.bfloat16)}
        if case["train"]:
            x["do"] = _randn((B * T, F), gen, torch.bfloat16)
        return x
    if op == "write":
        k, v = _keys_values(case["B"], case["T"], case["H"], case["D"], gen, _DTYPES[case["dtype"]])
        return {"k": k, "v": v, "counts": torch.tensor(_counts(case), dtype=torch.int32, device="cuda")}
    if op == "attend":
        dt = _DTYPES[case["dtype"]]
        k, v = _keys_values(case["B"], case["keys"], case["Hkv"], case["D"], gen, dt)
        q = _randn((case["B"], case["Tq"], case["Hq"], case["D"]), gen, dt)
        return {"k": k, "v": v, "q": q, "lens": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")}
    x = {"logits": _logits(case, gen), "u": torch.rand((case["rows"],), generator=gen, device="cuda")}
    names = ("temperature", "top_k", "top_p", "min_p")
    if case["per_row"]:
        r = torch.rand((4, case["rows"]), generator=gen, device="cuda")
        x["temperature"] = (case["temperature"] * (0.5 + r[0])).float()
        x["top_k"] = (case["top_k"] * (r[1] > 0.3) * (0.5 + r[1])).to(torch.int32)
        x["top_p"] = torch.where(r[2] > 0.3, torch.full_like(r[2], case["top_p"]), torch.ones_like(r[2]))
        x["min_p"] = (case["min_p"] * (r[3] > 0.3)).float()
    else:
        x.update({n: case[n] for n in names})
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    op = case["op"]
    state = {"case": case}
    if op == "write":
        state.update(x)
        cap = case["start"] + case["T"]
        if own:
            from underhfs_b200.kv_cache import QuantizedKVCache

            cache = QuantizedKVCache(1, case["B"], case["H"], case["D"], cap, device="cuda")
            cache.advance(case["start"])
            state["cache"] = cache
        else:
            state["cache"] = {n: _empty_plain(case["B"], cap, case["H"], case["D"]) for n in "kv"}
        return state
    if op == "attend":
        state["q"] = x["q"]
        if own:
            from underhfs_b200.kv_cache import QuantizedKVCache

            cache = QuantizedKVCache(1, case["B"], case["Hkv"], case["D"], case["keys"], device="cuda")
            cache.append(0, x["k"], x["v"], counts=x["lens"])
            cache.advance(x["lens"] - case["Tq"])
            state["cache"] = cache
        else:
            state["lens"] = _lengths(case)
            for n in "kv":
                state[n] = [_quantize(x[n][b : b + 1]) for b in range(case["B"])]
        return state
    state.update(x)
    return state


# --------------------------------------------------------- the plain form: cache
def _quantize(x):
    """x [..., D] -> (codes [..., D/2] uint8 with two codes to a byte, s, lo [..., D/32] fp16)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo = g.amin(-1).clamp(-65504.0, 65504.0).half()
    s = ((g.amax(-1) - lo.float()) / 15.0).clamp(max=65504.0).half()
    # in 64 bits: a quotient next to a half has to fall on its own side
    d, sd = g.double() - lo.double().unsqueeze(-1), s.double().unsqueeze(-1)
    c = torch.round(d / torch.where(sd > 0, sd, torch.full_like(sd, math.inf)))
    c = c.clamp(0, 15).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), s, lo


def _dequantize(packed, s, lo):
    c = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (lo.float().unsqueeze(-1) + s.float().unsqueeze(-1) * c).flatten(-2)


def _empty_plain(B, cap, H, D):
    z = dict(device="cuda")
    return [torch.zeros((B, cap, H, D // 2), dtype=torch.uint8, **z),
            torch.zeros((B, cap, H, D // GROUP), dtype=torch.float16, **z),
            torch.zeros((B, cap, H, D // GROUP), dtype=torch.float16, **z)]


def _write_plain(state):
    case = state["case"]
    start, T = case["start"], case["T"]
    live = torch.arange(T, device="cuda").unsqueeze(0) < state["counts"].unsqueeze(1)  # [B, T]
    out = []
    for n in "kv":
        store = state["cache"][n]
        for old, new in zip(store, _quantize(state[n])):
            part = old[:, start : start + T]
            part.copy_(torch.where(live[:, :, None, None], new, part))
        out.append(_dequantize(*[t[:, start : start + T] for t in store]).to(_DTYPES[case["dtype"]]))
    return tuple(out)


def _visible(qpos, kpos, window, sinks):
    ok = kpos <= qpos
    if window:
        ok = ok & ((qpos - kpos < window) | (kpos < sinks))
    return ok


def _attend_plain(state):
    case = state["case"]
    q, Tq, D, G = state["q"], case["Tq"], case["D"], case["Hq"] // case["Hkv"]
    out = torch.empty_like(q)
    for b, n in enumerate(state["lens"]):
        k, v = ([t[0, :n] for t in state[x][b]] for x in "kv")
        k, v = _dequantize(*k).transpose(0, 1), _dequantize(*v).transpose(0, 1)  # [Hkv, n, D]
        qb = q[b].float().view(Tq, case["Hkv"], G, D).permute(1, 2, 0, 3).reshape(case["Hkv"], G * Tq, D)
        s = (qb @ k.transpose(1, 2)) / math.sqrt(D)
        pos = torch.arange(n, device="cuda")
        ok = _visible(pos[n - Tq :].unsqueeze(1), pos.unsqueeze(0), case["window"], case["sinks"])
        s = s.view(-1, G, Tq, n).masked_fill(~ok, -math.inf).view(-1, G * Tq, n)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
        out[b] = o.view(case["Hkv"], G, Tq, D).permute(2, 0, 1, 3).reshape(Tq, case["Hq"], D).to(q.dtype)
    return out


# ---------------------------------------------------- the plain form: training
def _window_plain(state):
    case = state["case"]
    B, T, H, D = (case[n] for n in "BTHD")
    scale = 1.0 / math.sqrt(D)
    q, k, v = state["qkv"].view(B, T, 3, H, D).permute(2, 0, 3, 1, 4)
    pos = torch.arange(T, device="cuda")
    hide = ~_visible(pos.unsqueeze(1), pos.unsqueeze(0), case["window"], case["sinks"])
    o = torch.empty((B, T, H, D), dtype=torch.bfloat16, device="cuda")
    grad = torch.empty((B, T, 3, H, D), dtype=torch.bfloat16, device="cuda") if case["train"] else None
    step = max(1, min(H, (1 << 28) // (T * T)))  # heads at once: a score matrix of 1 GB at most
    for b in range(B):
        for h in range(0, H, step):
            part = slice(h, min(H, h + step))
            qf, kf, vf = (t[b, part].float() for t in (q, k, v))
            p = (qf @ kf.transpose(1, 2)) * scale
            p.masked_fill_(hide, -math.inf)
            p.sub_(p.amax(-1, keepdim=True)).exp_()
            p /= p.sum(-1, keepdim=True)
            of = p @ vf
            o[b, :, part] = of.transpose(0, 1).to(o.dtype)
            if grad is None:
                continue
            do = state["do"].view(B, T, H, D)[b, :, part].transpose(0, 1).float()
            dv = p.transpose(1, 2) @ do
            ds = do @ vf.transpose(1, 2)
            ds.sub_((do * of).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            for i, g in enumerate((ds @ kf, ds.transpose(1, 2) @ qf, dv)):
                grad[b, :, i, part] = g.transpose(0, 1).to(grad.dtype)
    o = o.view(B * T, H * D)
    return o if grad is None else (o, grad.view(B * T, 3 * H * D))


# ---------------------------------------------------- the plain form: sampling
def _column(value, rows):
    t = value if torch.is_tensor(value) else torch.full((rows,), float(value), dtype=torch.float64, device="cuda")
    return t.double().unsqueeze(1)


def _sample_plain(state):
    x = state["logits"].double()
    rows, vocab = x.shape
    temp, top_k, top_p, min_p = (_column(state[n], rows) for n in ("temperature", "top_k", "top_p", "min_p"))
    # sorted by value, equal values by index
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((val - val[:, :1]) / torch.where(temp > 0, temp, torch.ones_like(temp)))
    rank = torch.arange(vocab, device="cuda").unsqueeze(0)
    keep = (rank < torch.where(top_k > 0, top_k, torch.full_like(top_k, vocab))) & (val > -math.inf)
    w = w * keep
    before = torch.cumsum(w, 1) - w
    keep = keep & ((top_p >= 1.0) | (before < top_p * w.sum(1, keepdim=True))) & (w >= min_p)
    # in the order of the vocabulary: the first token whose running sum passes u times the whole
    kept = torch.zeros_like(w).scatter_(1, idx, w * keep)
    run_sum = torch.cumsum(kept, 1)
    goal = state["u"].double().unsqueeze(1) * run_sum[:, -1:]
    token = (run_sum <= goal).sum(1)
    return torch.where(temp[:, 0] > 0, token, idx[:, 0])


# ------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"window": _window_plain, "write": _write_plain, "attend": _attend_plain, "sample": _sample_plain}[op](
            state)
    if op == "window":
        from underhfs_b200.ops.functions import flash_attention

        B, T, H, D = (case[n] for n in "BTHD")
        if not case["train"]:
            with torch.no_grad():
                return flash_attention(state["qkv"], B, T, H, D, True, window=case["window"], sinks=case["sinks"])
        qkv = state["qkv"].detach().requires_grad_(True)
        o = flash_attention(qkv, B, T, H, D, True, window=case["window"], sinks=case["sinks"])
        (dqkv,) = torch.autograd.grad(o, qkv, state["do"])
        return o.detach(), dqkv
    if op == "write":
        cache = state["cache"]
        cache.append(0, state["k"], state["v"], counts=state["counts"] if case["ragged"] else None)
        return cache.read(0, case["start"], case["T"], dtype=_DTYPES[case["dtype"]])
    if op == "attend":
        return state["cache"].attend(0, state["q"], window=case["window"] or None, sinks=case["sinks"])
    from underhfs_b200 import functional as F

    return F.sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                    top_p=state["top_p"], min_p=state["min_p"]).torch()


# ------------------------------------------------------------------------ work
def _pairs(T, window, sinks, first=0):
    """Visible (query, key) pairs of queries first..T-1."""
    n = 0
    for i in range(first, T):
        n += i + 1 if not window else min(i + 1, window + min(sinks, max(0, i + 1 - window)))
    return n


def _keys_seen(n, tq, window, sinks):
    """Keys of a sequence of n that at least one of its last tq tokens sees."""
    if not window:
        return n
    lo = max(0, n - tq - window + 1)
    return n - lo + min(sinks, lo)


def work(case):
    op, D = case["op"], case.get("D", 0)
    row = D // 2 + (D // GROUP) * 4  # bytes of one key (or value) of one head in the cache
    if op == "window":
        B, T, H = case["B"], case["T"], case["H"]
        el = B * T * H * D
        flops = 4.0 * B * H * D * _pairs(T, case["window"], case["sinks"])
        if not case["train"]:
            return {"bytes": 2 * 4 * el, "flops": flops}
        # backward: S again, dP, dV, dQ, dK
        return {"bytes": 2 * (4 + 1 + 3) * el, "flops": flops * 3.5}
    if op == "write":
        n = sum(_counts(case)) * case["H"]
        full = case["B"] * case["T"] * case["H"]
        el = _BYTES[case["dtype"]]
        return {"bytes": 2 * (n * (D * el + row) + full * (row + D * el)), "flops": 2.0 * (n * 6 * D + full * 2 * D)}
    if op == "attend":
        lens, tq = _lengths(case), case["Tq"]
        seen = sum(_keys_seen(n, tq, case["window"], case["sinks"]) for n in lens)
        pairs = sum(_pairs(n, case["window"], case["sinks"], n - tq) for n in lens)
        return {"bytes": 2 * seen * case["Hkv"] * row + 4 * case["B"] * tq * case["Hq"] * D,
                "flops": 4.0 * pairs * case["Hq"] * D}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * _BYTES[case["dtype"]] + 12 * case["rows"], "flops": 8.0 * n}


# ----------------------------------------------------------------------- exact
def _exact_groups(x):
    """The values that the 4-bit codes of x [n, 32] (64 bits) stand for."""
    lo = torch.min(x, 1).values.clamp(-65504.0, 65504.0).to(torch.float32).to(torch.float16).double()
    s = ((torch.max(x, 1).values - lo).float() / 15.0).clamp(max=65504.0).half().double()
    lo, s = lo[:, None], s[:, None]
    code = torch.where(s > 0, ((x - lo) / torch.where(s > 0, s, torch.ones_like(s))).round(), torch.zeros_like(x))
    return lo + s * torch.clamp(code, 0.0, 15.0)


def _exact_values(x):
    return _exact_groups(x.double().reshape(-1, GROUP)).reshape(x.shape)


def _exact_attention(q, k, v, ok):
    """q [.., m, D], k, v [.., n, D], ok [m, n]."""
    s = torch.einsum("...md,...nd->...mn", q, k) * q.shape[-1] ** -0.5
    return torch.einsum("...mn,...nd->...md", torch.softmax(s.masked_fill(~ok, float("-inf")), -1), v)


def _exact_mask(first, n, window, sinks):
    i, j = torch.meshgrid(torch.arange(first, n, device="cuda"), torch.arange(n, device="cuda"), indexing="ij")
    ok = i >= j
    return ok if not window else ok & torch.logical_or(j < sinks, j > i - window)


def exact(case, seed):
    x = _inputs(case, seed)
    op = case["op"]
    if op == "window":
        B, T, H, D = (case[n] for n in "BTHD")
        ok = _exact_mask(0, T, case["window"], case["sinks"])
        o = torch.empty((B, T, H, D), dtype=torch.float64, device="cuda")
        g = torch.empty((B, T, 3, H, D), dtype=torch.float64, device="cuda")
        for b in range(B):
            for h in range(H):
                part = x["qkv"].view(B, T, 3, H, D)[b, :, :, h].double().requires_grad_(case["train"])
                y = _exact_attention(part[:, 0], part[:, 1], part[:, 2], ok)
                o[b, :, h] = y.detach()
                if case["train"]:
                    y.backward(x["do"].view(B, T, H, D)[b, :, h].double())
                    g[b, :, :, h] = part.grad
        o = o.view(B * T, H * D)
        return (o, g.view(B * T, 3 * H * D)) if case["train"] else o
    if op == "write":
        out = []
        for n in "kv":
            y = torch.zeros(x[n].shape, dtype=torch.float64, device="cuda")
            for b, c in enumerate(_counts(case)):
                y[b, :c] = _exact_values(x[n][b, :c])
            out.append(y)
        return tuple(out)
    if op == "attend":
        Hkv, D, Tq = case["Hkv"], case["D"], case["Tq"]
        out = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(case)):
            ok = _exact_mask(n - Tq, n, case["window"], case["sinks"])
            for h in range(Hkv):
                k, v = (_exact_values(x[t][b, :n, h]) for t in "kv")
                heads = slice(h * (case["Hq"] // Hkv), (h + 1) * (case["Hq"] // Hkv))
                q = x["q"][b, :, heads].double().transpose(0, 1)
                out[b, :, heads] = _exact_attention(q, k, v, ok).transpose(0, 1)
        return out
    rows = case["rows"]
    tokens = torch.empty((rows,), dtype=torch.int64, device="cuda")
    for r in range(rows):
        z = x["logits"][r].double()
        t, k, p, m = (float(x[n][r]) if torch.is_tensor(x[n]) else float(x[n])
                      for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            tokens[r] = torch.nonzero(z == z.max())[0, 0]
            continue
        order = torch.argsort(-z, stable=True)
        order = order[torch.isfinite(z[order])]
        if k > 0:
            order = order[: int(k)]
        prob = torch.softmax(z[order] / t, 0)
        n = int((torch.cumsum(prob, 0) - prob < p).sum()) if p < 1.0 else len(order)
        n = min(n, int((prob >= m * prob[0]).sum()))
        left = torch.sort(order[:n]).values
        part = torch.cumsum(torch.softmax(z[left] / t, 0), 0)
        tokens[r] = left[min(int((part <= float(x["u"][r]) * part[-1]).sum()), n - 1)]
    return tokens
