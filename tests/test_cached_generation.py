"""TransformerLM.decode / generate over the 4-bit cache with sampling: the operators as they are used together."""

import json

import pytest
import torch

from underhfs import functional as F
from underhfs.cli import main
from underhfs.nn import TransformerLM
from underhfs.tensor import tensor

KW = dict(vocab_size=64, max_seq_len=48, features=64, hidden_features=96, layers=2, heads=2, init="normal", seed=3)


def lm(**kw):
    return TransformerLM(**{**KW, **kw})


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("window,sinks", [(None, 0), (6, 2)])
def test_cpu_prompt_is_exact_and_steps_follow_closely(window, sinks):
    m = lm(window=window, sinks=sinks)
    ids = torch.randint(0, 64, (2, 12), generator=torch.Generator().manual_seed(0))
    cache = m.new_cache(batch=2, max_len=20)
    with torch.no_grad():
        full = m(ids)._data
    got = m.decode(ids[:, :9], cache)._data
    assert torch.allclose(got, full[:, 8], rtol=0, atol=1e-12)
    for t in range(9, 12):  # over the quantised cache: near, not equal
        got = m.decode(ids[:, t : t + 1], cache)._data
        assert 0 < (got - full[:, t]).norm() < 0.05 * full[:, t].norm()
    assert cache.lengths.tolist() == [12, 12] and not cache.is_empty


def test_cpu_ragged_prompts_match_single_ones():
    m = lm()
    ids = torch.randint(0, 64, (2, 10), generator=torch.Generator().manual_seed(1))
    counts = torch.tensor([10, 4])
    cache = m.new_cache(batch=2)
    got = [m.decode(ids, cache, counts)._data, m.decode(ids[:, :2], cache)._data]
    assert cache.lengths.tolist() == [12, 6]
    for b, n in enumerate(counts.tolist()):
        one = m.new_cache()
        want = [m.decode(ids[b : b + 1, :n], one)._data, m.decode(ids[b : b + 1, :2], one)._data]
        for g, w in zip(got, want):
            assert torch.allclose(g[b], w[0], rtol=0, atol=1e-12)


def test_cpu_lengths_written_directly_are_seen():
    """`lengths` is the caller's to write (to go back to an earlier state, say): what is kept is attended to."""
    m = lm()
    ids = torch.randint(0, 64, (1, 12), generator=torch.Generator().manual_seed(3))
    cache = m.new_cache(max_len=20)
    first = m.decode(ids[:, :9], cache)._data
    held = cache.lengths.clone()
    want = m.decode(ids[:, 9:10], cache)._data
    cache.reset()
    assert cache.is_empty
    cache.lengths.copy_(held)
    assert not cache.is_empty
    assert torch.equal(m.decode(ids[:, 9:10], cache)._data, want)
    cache.lengths.zero_()
    assert cache.is_empty
    assert torch.equal(m.decode(ids[:, :9], cache)._data, first)
    cache.lengths = held * 0
    assert cache.is_empty
    cache.lengths = held.clone()
    assert torch.equal(m.decode(ids[:, 9:10], cache)._data, want)


def test_cpu_cache_made_in_inference_mode():
    m = lm()
    ids = torch.randint(0, 64, (1, 6), generator=torch.Generator().manual_seed(3))
    with torch.inference_mode():
        cache = m.new_cache(max_len=20)
        m.decode(ids[:, :4], cache)
        assert not cache.is_empty
    m.decode(ids[:, 4:], cache)
    assert cache.lengths.tolist() == [6]


def counts_outside_their_range(m, device):
    """A sequence brings between none and all of the T new tokens, whatever its count says: no row of
    another sequence, or of none, is taken for its last one, and the lengths stay true."""
    ids = torch.randint(0, 64, (3, 6), generator=torch.Generator().manual_seed(3)).to(device)
    held = lambda *v: torch.tensor(v, device=device)  # noqa: E731
    a, b = m.new_cache(batch=3), m.new_cache(batch=3)
    for part, counts, same in ((ids[:, :4], (4, -2, 7), (4, 0, 4)), (ids[:, 4:], (2**33 + 1, 2, 1), (2, 2, 1))):
        got = m.decode(part, a, held(*counts))._data
        want = m.decode(part, b, held(*same))._data
        assert torch.equal(got[[0, 2]], want[[0, 2]])
        assert a.lengths.tolist() == b.lengths.tolist()
    assert a.lengths.tolist() == [6, 2, 5]
    assert torch.equal(m.decode(ids[:, :1], a)._data, m.decode(ids[:, :1], b, tensor([1, 1, 1]).torch().long().to(device))._data)


def test_cpu_counts_outside_their_range():
    counts_outside_their_range(lm(), "cpu")


def past_the_end(m, device):
    """Ragged sequences: the step that does not fit is refused and leaves the cache as it was."""
    ids = torch.randint(0, 64, (2, 6), generator=torch.Generator().manual_seed(3)).to(device)
    held = lambda *v: torch.tensor(v, device=device)  # noqa: E731
    cache = m.new_cache(batch=2, max_len=10)
    m.decode(ids, cache, held(6, 3))
    for _ in range(4):
        m.decode(ids[:, :1], cache)
    for counts in (None, held(1, 0), held(2, 2)):
        with pytest.raises(ValueError, match="do not fit"):
            m.decode(ids[:, :1 if counts is None else 2], cache, counts)
        assert cache.lengths.tolist() == [10, 7]
    m.decode(ids[:, :4], cache, held(0, 2))  # (padded beyond the end, but what counts fits)
    assert cache.lengths.tolist() == [10, 9]
    with pytest.raises(ValueError, match="do not fit"):
        m.decode(ids[:, :1], cache)
    cache.lengths.copy_(torch.tensor([3, 9], dtype=torch.int32))
    m.decode(ids[:, :1], cache)
    with pytest.raises(ValueError, match="do not fit"):
        m.decode(ids[:, :1], cache)
    cache.reset()
    m.decode(ids, cache)
    assert cache.lengths.tolist() == [6, 6]


def test_cpu_past_the_end_of_ragged_sequences():
    past_the_end(lm(), "cpu")


def test_generate_samples_and_defaults_to_greedy():
    m = lm()
    prompt = tensor([1, 2, 3])
    greedy = m.generate(prompt, 6)._storage
    assert greedy == m.generate(prompt, 6, temperature=0.0)._storage
    assert greedy == m.generate(prompt, 6, temperature=2.0, top_k=1, seed=0)._storage
    a, b = (m.generate(prompt, 30, temperature=2.0, seed=5)._storage for _ in range(2))
    assert a == b and a != m.generate(prompt, 30, temperature=2.0, seed=6)._storage
    u = torch.rand(4, generator=torch.Generator().manual_seed(2))
    ids = [1, 2, 3]
    for i in range(4):
        with torch.no_grad():
            logits = m(torch.tensor(ids))._data[-1]
        ids.append(int(F.sample(logits, u[i].double(), temperature=1.5, top_p=0.9).torch()))
    assert m.generate(prompt, 4, temperature=1.5, top_p=0.9, uniform=u)._storage == ids


def test_generate_over_the_cache_on_the_cpu():
    m = lm()
    prompt = tensor([5, 6, 7, 8])
    out = m.generate(prompt, 8, cache="int4")._storage
    assert len(out) == 12 and out[:5] == m.generate(prompt, 1)._storage  # the first token comes from exact keys
    cache = m.new_cache(max_len=40)
    for _ in range(2):  # a cache is reset and used again
        assert m.generate(prompt, 8, cache=cache)._storage == out
    assert m.generate(prompt, 0, cache="int4")._storage == [5, 6, 7, 8]


@pytest.mark.parametrize("cache", [None, "int4"])
@pytest.mark.parametrize("kw,match", [
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(top_p=7.0), "top_p"), (dict(top_p=-0.5), "top_p"), (dict(top_k=-3), "top_k"), (dict(min_p=2.0), "min_p"),
    (dict(temperature=0.5, min_p=float("nan")), "min_p")])
@pytest.mark.parametrize("n", [0, 3])
def test_generate_refuses_settings_with_and_without_a_cache(kw, match, cache, n):
    """Greedy decoding uses none of them, but a wrong one is refused all the same."""
    with pytest.raises(ValueError, match=match):
        lm().generate(tensor([1, 2]), n, cache=cache, **kw)


def test_a_refused_generate_leaves_the_cache_as_it_was():
    m = lm()
    ids = torch.randint(0, 64, (1, 9), generator=torch.Generator().manual_seed(3))
    cache, other = m.new_cache(max_len=20), lm(layers=1).new_cache(max_len=30)
    pair = m.new_cache(batch=2, max_len=20)
    m.decode(ids, cache)
    want = cache.read(0, 0, 9, dtype=torch.float64)[0].clone()
    lm(layers=1).decode(ids, other)
    pair.advance(4)
    for c, prompt, n, match in ((cache, [1] * 15, 6, "do not fit"), (cache, [], 2, "prompt"), (other, [1, 2], 3, "another model"),
                                (pair, [1, 2], 3, "token ids")):
        with pytest.raises(ValueError, match=match):
            m.generate(torch.tensor(prompt, dtype=torch.int64), n, cache=c)
    assert cache.lengths.tolist() == [9] and other.lengths.tolist() == [9] and pair.lengths.tolist() == [4, 4]
    assert torch.equal(cache.read(0, 0, 9, dtype=torch.float64)[0], want)


def no_token_to_choose(m, kw):
    with torch.no_grad():
        m.norm.weight._data.fill_(float("nan"))  # logits of NaN
    for cache in (None, "int4"):
        with pytest.raises(ValueError, match="no token"):
            m.generate(tensor([1, 2]), 9, cache=cache, temperature=0.7, **kw)
    with pytest.raises(ValueError, match="no token"):
        m.generate(tensor([1, 2]), 1, cache="int4")


def test_cpu_generate_without_a_token_to_choose():
    no_token_to_choose(lm(), {})
    no_token_to_choose(lm(), dict(top_k=3, top_p=0.9))


def test_only_causal_attention_decodes():
    from underhfs.kv_cache import QuantizedKVCache
    from underhfs.nn import SelfAttention

    cache = QuantizedKVCache(1, 1, 1, 32, 8, device="cpu")
    with pytest.raises(ValueError, match="causal"):
        SelfAttention(32).decode(tensor(torch.zeros(1, 2, 32)), cache, 0)
    assert (cache.read(0)[0] == 0).all()


def test_refusals():
    m = lm()
    with pytest.raises(ValueError, match="do not fit"):
        m.generate(tensor([1] * 40), 9, cache="int4")
    with pytest.raises(ValueError, match="unknown cache"):
        m.generate(tensor([1]), 2, cache="int8")
    with pytest.raises(ValueError, match="prompt"):
        m.generate(torch.zeros(0, dtype=torch.int64), 2, cache="int4")
    with pytest.raises(ValueError, match="uniform needs"):
        m.generate(tensor([1]), 3, temperature=1.0, uniform=torch.rand(2))
    with pytest.raises(ValueError, match="temperature"):
        m.generate(tensor([1]), 3, temperature=float("inf"))
    with pytest.raises(ValueError, match="another model"):
        m.decode(torch.zeros(1, 1, dtype=torch.int64), lm(layers=1).new_cache())
    with pytest.raises(ValueError, match="token ids"):
        m.decode(torch.zeros(2, 1, dtype=torch.int64), m.new_cache())
    with pytest.raises(ValueError, match="positions"):
        m.decode(torch.zeros(1, 1, dtype=torch.int64), lm(max_seq_len=99).new_cache())
    with pytest.raises(ValueError, match="head_dim"):
        lm(heads=8).new_cache()  # 8 channels a head: less than one group


def test_cli_generates_with_a_cache_and_sampling(capsys):
    args = ["generate", "--prompt", "hi", "--max-new-tokens", "5", "--features", "32", "--seq-len", "16",
            "--cache", "int4", "--temperature", "0.9", "--top-k", "20", "--top-p", "0.95", "--min-p", "0.01", "--seed", "4",
            "--window", "4", "--sinks", "1"]
    outs = []
    for _ in range(2):
        assert main(args) == 0
        outs.append(json.loads(capsys.readouterr().out)["tokens"])
    assert outs[0] == outs[1] and len(outs[0]) == 7


# ------------------------------------------------------------------- GPU
@pytest.fixture
def status_ok():
    yield
    from underhfs_b200.ops._lib import core

    st = core().device_status(True)
    assert st["code"] == 0, st


def gpu_pair(**kw):
    big = dict(vocab_size=512, max_seq_len=320, features=256, hidden_features=512, layers=3, heads=4, init="normal", seed=2)
    cpu, gpu = TransformerLM(**{**big, **kw}), TransformerLM(**{**big, **kw}).to("cuda", dtype="bf16")
    for (_, a), (_, b) in zip(cpu.named_parameters(), gpu.named_parameters()):
        with torch.no_grad():
            a._data.copy_(8 * b._data.double().cpu())  # larger weights: logits that differ
            b._data.copy_(a._data)
    return cpu, gpu


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [2, 4])  # head_dim 128, 64
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_engine_decodes_over_the_cache(heads, window, sinks, status_ok):
    """Ragged prompts, a chunk and single tokens: the prompt's logits are the plain forward's,
    and in every layer the step's keys, values and attention are what the formulas give for
    that layer's own input.  (Logits of different roundings are not compared: with these
    weights the plain bf16 forward alone is a quarter of their size from 64 bits.)"""
    from tests.test_kv_cache import check_attend
    from underhfs_b200.kv_cache import QuantizedKVCache, quantize_groups

    seen = []

    class Watched(QuantizedKVCache):
        def append(self, layer, k, v, counts=None):
            super().append(layer, k, v, counts=counts)
            at, n = self.lengths.tolist(), [k.shape[1]] * self.batch if counts is None else counts.tolist()
            for x, got in zip((k, v), self.read(layer, dtype=torch.float32)):
                for b in range(self.batch):
                    assert torch.equal(got[b, at[b] : at[b] + n[b]], quantize_groups(x[b, : n[b]]).float())

        def attend(self, layer, q, **kw):
            o = super().attend(layer, q, **kw)
            one = QuantizedKVCache(1, self.batch, self.kv_heads, self.head_dim, self.max_len)
            one.pages = self.pages[layer : layer + 1]
            new = [q.shape[1]] * self.batch
            check_attend(one, q, o, [a + n for a, n in zip(self.lengths.tolist(), new)], new, window, sinks)
            seen.append(layer)
            return o

    _, gpu = gpu_pair(heads=heads, window=window, sinks=sinks)
    ids = torch.randint(0, 512, (2, 200), generator=torch.Generator().manual_seed(4)).cuda()
    counts = torch.tensor([150, 97], dtype=torch.int32, device="cuda")
    cache = Watched(3, 2, heads, 256 // heads, 300)
    got = gpu.decode(ids[:, :150], cache, counts)._data
    with torch.no_grad():
        full = gpu(ids[:, :150])._data
    assert torch.equal(got, torch.stack((full[0, 149], full[1, 96])))
    for x in (ids[:, 150:163], ids[:, 163:164], ids[:, 164:165]):
        assert gpu.decode(x, cache)._data.isfinite().all()
    assert seen == [0, 1, 2] * 3
    assert cache.lengths.tolist() == [165, 112]


@pytest.mark.gpu
def test_engine_steps_stay_near_the_whole_context(status_ok):
    """Weights of ordinary size: tokens run one by one over the cache against the whole context at once.

    The cache moves a value by at most 1/30 of its group's range (about 0.13 of a
    standard deviation; a third of that in the mean), a bf16 forward adds a few 2^-8:
    logits off by well under a tenth, those of another context by about their size.
    """
    kw = dict(vocab_size=512, max_seq_len=320, features=256, hidden_features=512, layers=3, heads=4, init="normal", seed=2)
    gpu = TransformerLM(**kw).to("cuda", dtype="bf16")
    ids = torch.randint(0, 512, (1, 100), generator=torch.Generator().manual_seed(4)).cuda()
    cache = gpu.new_cache()
    gpu.decode(ids[:, :60], cache)
    with torch.no_grad():
        full = gpu(ids)._data[0].double()
    for t in range(60, 100):
        got = gpu.decode(ids[:, t : t + 1], cache)._data[0].double()
        assert (got - full[t]).norm() < 0.1 * full[t].norm()
        assert (got - full[t - 1]).norm() > 0.5 * full[t].norm()


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)])
def test_generate_graph_equals_eager_steps(kw, status_ok):
    _, m = gpu_pair(window=64, sinks=4)
    prompt = list(range(3, 70))
    n = 60
    u = torch.rand(n, generator=torch.Generator().manual_seed(8))
    got = m.generate(tensor(prompt), n, cache="int4", uniform=u, **kw)._storage
    cache = m.new_cache()
    ids, out = torch.tensor([prompt], device="cuda"), []
    settings = {"temperature": 0.0, **kw}
    for i in range(n):
        tok = F.sample(m.decode(ids, cache)._data, u[i : i + 1].cuda(), **settings).torch()
        ids = tok.view(1, 1)
        out.append(int(tok))
    assert got == prompt + out
    # a second run on the same cache, and the uncached path still runs
    assert m.generate(tensor(prompt), n, cache=cache, uniform=u, **kw)._storage == got
    assert m.generate(tensor(prompt), 3, uniform=u[:3], **kw)._storage[: len(prompt) + 1] == got[: len(prompt) + 1]


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [0, 20])
def test_captured_steps_and_eager_ones_mix(prompt, status_ok):
    """Steps captured on an empty cache, reset, replayed (after an eager prompt or from nothing) and
    followed by eager calls: those see what the replays cached.  (The bounds are those of
    test_engine_steps_stay_near_the_whole_context.)"""
    kw = dict(vocab_size=512, max_seq_len=320, features=256, hidden_features=512, layers=3, heads=4, init="normal", seed=2)
    gpu = TransformerLM(**kw).to("cuda", dtype="bf16")
    ids = torch.randint(0, 512, (1, 64), generator=torch.Generator().manual_seed(6)).cuda()
    with torch.no_grad():
        full = gpu(ids)._data[0].double()
    cache, token = gpu.new_cache(), ids[:, :1].clone()
    gpu.decode(token, cache)  # (warm)
    cache.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu.decode(token, cache)._data
    for _ in range(2):
        cache.reset()
        assert cache.is_empty
        if prompt:
            with torch.no_grad():
                want = gpu(ids[:, :prompt])._data[0, -1]
            assert torch.equal(gpu.decode(ids[:, :prompt], cache)._data[0], want)  # its own exact keys and values
        for t in range(prompt, 40):
            token.copy_(ids[:, t : t + 1])
            graph.replay()
            assert t == 0 or (out[0].double() - full[t]).norm() < 0.1 * full[t].norm()
        assert not cache.is_empty
        for t in (40, 41):
            got = gpu.decode(ids[:, t : t + 1], cache)._data[0].double()
            assert (got - full[t]).norm() < 0.1 * full[t].norm()
        assert cache.lengths.tolist() == [42]
    cache.set_host_length(42)
    assert not cache.is_empty
    with pytest.raises(ValueError, match="do not fit"):
        gpu.decode(torch.zeros(1, 279, dtype=torch.int64), cache)


@pytest.mark.gpu
def test_counts_outside_their_range(status_ok):
    counts_outside_their_range(lm(features=128).to("cuda", dtype="bf16"), "cuda")


@pytest.mark.gpu
def test_past_the_end_of_ragged_sequences(status_ok):
    past_the_end(lm(features=128).to("cuda", dtype="bf16"), "cuda")


@pytest.mark.gpu
def test_ragged_steps_do_not_wait_for_the_device(status_ok):
    """Room is counted on the host: lengths are read back only where a sequence may be at its end."""
    m = lm(features=128).to("cuda", dtype="bf16")
    ids = torch.randint(0, 64, (2, 6)).cuda()
    cache, counts = m.new_cache(batch=2), torch.tensor([6, 3], device="cuda")
    m.decode(ids, cache, counts)
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(5):
            m.decode(ids, cache, counts)
            m.decode(ids[:, :1], cache)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert cache.lengths.tolist() == [41, 23]


@pytest.mark.gpu
@pytest.mark.parametrize("other", ["allocates", "waits", "generates"])
def test_generate_beside_another_thread(other, status_ok):
    """The captured steps of one thread and what another does meanwhile leave each other alone."""
    import threading

    _, m = gpu_pair()
    x = torch.randn(64, 64, device="cuda")
    kw = dict(cache="int4", temperature=0.9, top_p=0.95)
    want = [m.generate(tensor([3, 1, 4]), 40, seed=s, **kw)._storage for s in range(6)]
    torch.cuda.synchronize()
    done, failed = threading.Event(), []

    def beside():
        n = 0
        try:
            while not done.is_set():
                n += 1
                if other == "allocates":
                    torch.empty(n % 61 + 1, 1 << 20, device="cuda")
                    if n % 50 == 0:
                        torch.cuda.empty_cache()
                elif other == "waits":
                    assert x.sum().item() is not None
                else:
                    assert m.generate(tensor([3, 1, 4]), 40, seed=n % 6, **kw)._storage == want[n % 6]
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    t = threading.Thread(target=beside)
    t.start()
    try:
        for _ in range(3):
            for s in range(6):
                assert m.generate(tensor([3, 1, 4]), 40, seed=s, **kw)._storage == want[s]
    finally:
        done.set()
        t.join()
    assert not failed, failed
    assert torch.randn(3, device="cuda").isfinite().all()
    assert torch.cuda.current_stream() == torch.cuda.default_stream()


@pytest.mark.gpu
def test_generate_without_a_token_to_choose():
    from underhfs_b200.ops._lib import core

    no_token_to_choose(lm(features=128).to("cuda", dtype="bf16"), {})
    core().device_status(True)  # the steps after it reported a token outside the vocabulary


@pytest.mark.gpu
def test_a_cache_on_another_device_is_refused_and_kept():
    m = lm(features=128).to("cuda", dtype="bf16")
    cache = lm(features=128).new_cache()
    cache.advance(5)
    for call in (lambda: m.decode(torch.zeros(1, 2, dtype=torch.int64), cache), lambda: m.generate(tensor([1]), 2, cache=cache)):
        with pytest.raises(RuntimeError, match="the cache is on cpu"):
            call()
    assert cache.lengths.tolist() == [5]


@pytest.mark.gpu
def test_cache_needs_the_engine_on_cuda():
    m = lm(features=64, heads=1).to("cuda")
    with pytest.raises(ValueError, match="bf16 engine"):
        m.new_cache()
