"""A key / value cache held in 4 bits, and attention over it.

The reference keeps no cache: its generate() runs the whole context again for
every token (nn.py:318-334).  ``QuantizedKVCache`` holds the keys and values
of every layer at 5 bits a value (4-bit codes and an fp16 scale and minimum for
each 32 channels of a token and head), so a token of decoding reads 0.31 of
the bytes of a bf16 cache:

    cache = QuantizedKVCache(layers, batch, kv_heads, head_dim, max_len, device="cuda")
    cache.append(layer, k, v)          # k, v [batch, tokens, kv_heads, head_dim]
    o = cache.attend(layer, q)         # q [batch, tokens, heads, head_dim]
    cache.advance(tokens)              # once every layer has the tokens

``append`` writes behind the tokens that ``advance`` has counted, so a step
that is not advanced (rejected drafts, a retried step) is simply written over.
On CUDA each call is one kernel of csrc/kernels/kv4.cu (head_dim 64 or 128); on
the CPU the same arithmetic runs in float64.
"""

from __future__ import annotations

import contextlib
import math

import torch

from underhfs_b200.ops import kernels as K

GROUP = 32   # channels that share a scale and a minimum
PAGE = 32    # tokens per page of the CUDA layout
RANGE = 61440.0  # values are held to +-RANGE, where lo + scale * code is a finite fp16 number


def _raw(t) -> torch.Tensor:
    return t if isinstance(t, torch.Tensor) else t._data


_HERE = contextlib.nullcontext()


def _no_inference_mode():
    return torch.inference_mode(False) if torch.is_inference_mode_enabled() else _HERE


def quantize_groups(x: torch.Tensor) -> torch.Tensor:
    """The values (float64) that the 4-bit codes of x [..., D] stand for.

    For each 32 channels: lo = fp16(min), s = fp16((max - lo) * fp32(1 / 15)),
    code = round-half-even((x - lo) / s) in 0..15 (0 where s is 0), value lo + s * code.
    Values beyond +-RANGE are held to it and NaN becomes the group's minimum.
    """
    g = x.double().unflatten(-1, (-1, GROUP))
    nan = torch.isnan(g)
    inf = torch.full_like(g, math.inf)
    lo = torch.where(nan, inf, g).amin(-1, keepdim=True)
    hi = torch.where(nan, -inf, g).amax(-1, keepdim=True)
    empty = lo > hi
    lo, hi = (torch.where(empty, torch.zeros_like(t), t).clamp(-RANGE, RANGE) for t in (lo, hi))
    lo = lo.float().half().double()
    s = ((hi - lo).float() * (1.0 / 15.0)).clamp(min=0).half().double()
    code = torch.round((torch.where(nan, lo, g) - lo) / torch.where(s > 0, s, inf[..., :1]))
    return (lo + s * code.clamp(0, 15)).flatten(-2)


class QuantizedKVCache:
    """Keys and values of ``layers`` layers and ``batch`` sequences of up to ``max_len`` tokens in 4 bits."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, max_len: int, *,
                 device: "str | torch.device" = "cuda") -> None:
        for name, value in (("layers", layers), ("batch", batch), ("kv_heads", kv_heads), ("max_len", max_len)):
            if int(value) < 1:
                raise ValueError(f"{name} must be at least 1, got {value}")
        self.device = torch.device(device)
        self._cuda = self.device.type == "cuda"
        self.layers, self.batch, self.kv_heads = int(layers), int(batch), int(kv_heads)
        self.head_dim, self.max_len = int(head_dim), int(max_len)
        if self._cuda and self.head_dim not in (64, 128):
            raise ValueError(f"the CUDA cache takes head_dim 64 or 128, got {head_dim}")
        if not self._cuda and (self.head_dim < GROUP or self.head_dim % GROUP):
            raise ValueError(f"head_dim must be a multiple of {GROUP}, got {head_dim}")
        with _no_inference_mode():  # inference tensors could not be written later, and count no versions
            if self._cuda:
                pages = (self.max_len + PAGE - 1) // PAGE
                self.pages = torch.zeros((self.layers, self.batch, self.kv_heads, pages, 40 * self.head_dim),
                                         dtype=torch.uint8, device=self.device)
                self.device = self.pages.device
            else:
                self._k, self._v = (torch.zeros((self.layers, self.batch, self.max_len, self.kv_heads, self.head_dim),
                                                dtype=torch.float64) for _ in range(2))
            self.lengths = torch.zeros((self.batch,), dtype=torch.int32, device=self.device)
        # A captured step changes the lengths at every replay, which the host does not see
        self._captured = False
        self._note(0, 0)

    @property
    def pages(self) -> torch.Tensor:
        """CUDA: the codes, scales and minima, uint8 [layers, batch, kv_heads, pages, 40 head_dim]."""
        return self._pages

    @pages.setter
    def pages(self, value: torch.Tensor) -> None:
        self._pages = value
        self._layer_pages = list(value)  # making a view costs as much as a launch

    @property
    def lengths(self) -> torch.Tensor:
        """Tokens of each sequence that ``advance`` has counted: int32 [batch], on the
        cache's device.  It may be written to, but not by a captured step (which takes ``advance``)."""
        return self._lengths

    @lengths.setter
    def lengths(self, value: torch.Tensor) -> None:
        if value.shape != (self.batch,) or value.dtype != torch.int32 or value.device != self.device:
            raise ValueError(f"lengths must be int32 [{self.batch}] on {self.device}, got {value.dtype} "
                             f"{list(value.shape)} on {value.device}")
        with _no_inference_mode():
            self._lengths = value.clone() if value.is_inference() else value.contiguous()
        self._version = -1

    # What the host knows of the lengths: their common value (None where they differ) and a number that
    # none passes (None: not known).  It holds for one version of the tensor, so writes from
    # outside are noticed.
    def _note(self, length: int | None, bound: int | None) -> None:
        self._host_length, self._host_bound = length, bound
        self._version = self._lengths._version

    def _known(self) -> bool:
        return not self._captured and self._version == self._lengths._version

    def _capturing(self) -> bool:
        return self._cuda and torch._C._cuda_isCurrentStreamCapturing()

    @property
    def nbytes(self) -> int:
        """Device bytes of the keys and values."""
        if self._cuda:
            return self.pages.numel()
        return self._k.element_size() * 2 * self._k.numel()

    @property
    def is_empty(self) -> bool:
        """No sequence has a token.  Reads the lengths back where the host cannot know them: after
        they were written to, or once a step with ``advance`` was captured.  False while
        a step is captured, since it may be replayed on any lengths."""
        if self._known():
            return self._host_length == 0 and not self._capturing()
        return not self._capturing() and not bool(self._lengths.any())

    # ------------------------------------------------------------- checks
    def _on_device(self):
        """Launch on the cache's device, whichever is current."""
        if not self._cuda or self.device.index == torch._C._cuda_getDevice():
            return _HERE
        return torch.cuda.device(self.device)

    def _check_layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} outside [0, {self.layers})")
        return layer

    def _check_counts(self, counts) -> torch.Tensor:
        counts = _raw(counts)
        if counts.shape != (self.batch,):
            raise ValueError(f"counts must have shape [{self.batch}], got {list(counts.shape)}")
        if counts.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"counts must be int32 or int64, got {counts.dtype}")
        if counts.device != self.device:
            raise RuntimeError(f"counts are on {counts.device}, the cache on {self.device}")
        if counts.dtype == torch.int32 and counts.is_contiguous():
            return counts
        return counts.clamp(-(2**31), 2**31 - 1).to(torch.int32).contiguous()  # (nothing wraps round)

    def _check_rows(self, t, name: str, heads: int | None) -> torch.Tensor:
        """t as [batch, tokens, heads (None: any), head_dim] on the cache's device."""
        if not isinstance(t, torch.Tensor):
            t = t._data
        shape = t.shape
        if len(shape) != 4 or shape[0] != self.batch or shape[3] != self.head_dim or (
                heads is not None and shape[2] != heads):
            want = f"[{self.batch}, tokens, {'heads' if heads is None else heads}, {self.head_dim}]"
            raise ValueError(f"{name} must be {want}, got {list(shape)}")
        if t.device != self.device:
            raise RuntimeError(f"{name} is on {t.device}, the cache on {self.device}")
        if not t.is_floating_point():
            raise TypeError(f"{name} must be a floating-point tensor, got {t.dtype}")
        return t

    def _check_room(self, tokens: int) -> None:
        used = (self._host_length or 0) if self._known() else 0
        if used + tokens > self.max_len:
            raise ValueError(f"{tokens} more tokens do not fit: {used} of {self.max_len} are used")

    def admit(self, tokens: int, counts=None) -> torch.Tensor | None:
        """For a model's step of `tokens` new tokens: ``counts`` as every call understands them (int32,
        between 0 and `tokens`), for ``append``, ``attend`` and ``advance``.

        Raises where they do not fit.  The lengths are read back for that only when the host's
        bound on them leaves it open (ragged sequences near the end, lengths written from
        outside), and never while a step is captured: what replays put past the end is
        left out and reported in the device status word."""
        if counts is not None:
            counts = self._check_counts(counts).clamp(0, tokens)
        bound = self._host_bound if self._known() else None
        if (bound is None or bound + tokens > self.max_len) and not self._capturing():
            held = self._lengths.tolist()
            new = [tokens] * self.batch if counts is None else counts.tolist()
            for used, n in zip(held, new):
                if used + n > self.max_len:
                    raise ValueError(f"{n} more tokens do not fit: {used} of {self.max_len} are used")
            if not self._captured:
                self._note(held[0] if len(set(held)) == 1 else None, max(held))
        return counts

    # --------------------------------------------------------------- calls
    def append(self, layer: int, k, v, counts=None) -> None:
        """Quantise k / v [batch, tokens, kv_heads, head_dim] (fp32, fp16 or bf16,
        any strides) into `layer` behind each sequence's ``lengths`` tokens.

        ``counts`` (int tensor [batch], on the cache's device): sequence b
        brings only its first counts[b] tokens; the rest is not written.  Lengths
        held on the device are checked there: tokens past ``max_len`` are left
        out and reported in the device status word."""
        self._check_layer(layer)
        k, v = self._check_rows(k, "k", self.kv_heads), _raw(v)
        tokens = k.shape[1]
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError(f"k and v differ: {list(k.shape)} {k.dtype}, {list(v.shape)} {v.dtype}")
        if v.device != self.device:
            raise RuntimeError(f"v is on {v.device}, the cache on {self.device}")
        if counts is not None:
            counts = self._check_counts(counts)
        else:
            self._check_room(tokens)
        if tokens == 0:
            return
        if self._cuda:
            with self._on_device():
                K.kv4_append(self._layer_pages[layer], k, v, self.lengths, counts, self.max_len)
            return
        k, v = k.detach(), v.detach()
        for b in range(self.batch):
            n = k.shape[1] if counts is None else max(0, min(int(counts[b]), k.shape[1]))
            at = int(self.lengths[b])
            if at + n > self.max_len:
                raise ValueError(f"{n} more tokens do not fit: {at} of {self.max_len} are used")
            self._k[layer, b, at : at + n] = quantize_groups(k[b, :n])
            self._v[layer, b, at : at + n] = quantize_groups(v[b, :n])

    def attend(self, layer: int, q, *, window: int | None = None, sinks: int = 0, scale: float | None = None,
               counts=None) -> torch.Tensor:
        """Attention of the new tokens over `layer`, whose ``append`` has their
        keys and values: q [batch, tokens, heads, head_dim] (bf16 or fp16 on CUDA;
        heads a multiple of kv_heads, which consecutive query heads share) ->
        the same shape.  Token t of sequence b is at position lengths[b] + t and
        sees the keys up to its own; with ``window``, of those the last
        ``window`` and the first ``sinks``.  Rows t >= counts[b] are zeros.  Tokens past
        ``max_len`` see the keys that are there and are reported in the device status word.  No gradients."""
        self._check_layer(layer)
        q = self._check_rows(q, "q", None)
        heads, tokens = q.shape[2], q.shape[1]
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads are not a multiple of {self.kv_heads} key / value heads")
        if counts is not None:
            counts = self._check_counts(counts)
        else:
            self._check_room(tokens)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        window, sinks = (0, 0) if window is None and sinks == 0 else K.window_args(self.max_len, True, window, sinks)
        if self._cuda:
            if q.dtype not in (torch.bfloat16, torch.float16):
                raise TypeError(f"q must be bf16 or fp16, got {q.dtype}")
            if tokens == 0:
                return torch.empty_like(q)
            with self._on_device():
                return K.kv4_attend(self._layer_pages[layer], q, self.lengths, counts, self.max_len, scale, window, sinks)
        q = q.detach()
        out = torch.zeros(q.shape, dtype=torch.float64)
        for b in range(self.batch):
            n = tokens if counts is None else max(0, min(int(counts[b]), tokens))
            for t in range(n):
                pos = int(self.lengths[b]) + t
                key = torch.arange(pos + 1)
                seen = key if not window else key[(pos - key < window) | (key < sinks)]
                kk, vv = (x[layer, b, seen].repeat_interleave(heads // self.kv_heads, 1) for x in (self._k, self._v))
                p = torch.softmax(torch.einsum("hd,nhd->hn", q[b, t].double(), kk) * scale, -1)
                out[b, t] = torch.einsum("hn,nhd->hd", p, vv)
        return out.to(q.dtype)

    def read(self, layer: int, start: int = 0, count: int | None = None, *, dtype: torch.dtype = torch.bfloat16):
        """(k, v) [batch, count, kv_heads, head_dim]: what the cache's places
        start .. start + count - 1 stand for (to ``max_len`` by default), advanced
        or not; a place that was never written reads as 0."""
        self._check_layer(layer)
        count = self.max_len - start if count is None else count
        if start < 0 or count < 0 or start + count > self.max_len:
            raise ValueError(f"tokens {start}..{start + count - 1} are outside [0, {self.max_len})")
        if dtype not in (torch.float32, torch.float16, torch.bfloat16, torch.float64):
            raise TypeError(f"unsupported dtype {dtype}")
        if self._cuda:
            if dtype == torch.float64:
                raise TypeError("the CUDA cache reads as fp32, fp16 or bf16")
            with self._on_device():
                return K.kv4_read(self._layer_pages[layer], start, count, self.head_dim, dtype)
        return tuple(x[layer, :, start : start + count].to(dtype) for x in (self._k, self._v))

    def advance(self, tokens, *, at_most: int | None = None) -> None:
        """Count the appended tokens as part of the sequences: a number for all, or an int tensor
        [batch], of which the caller may know that none is above ``at_most``."""
        if isinstance(tokens, int):
            if tokens < 0:
                raise ValueError(f"tokens must not be negative, got {tokens}")
            self._check_room(tokens)
            length, at_most = self._host_length, tokens
        else:
            tokens, length = self._check_counts(tokens), None
        known, bound = self._known(), self._host_bound
        with self._on_device():
            self._lengths += tokens
        if self._capturing():
            self._captured = True  # replays count too
        elif known:
            self._note(None if length is None else length + tokens,
                       None if bound is None or at_most is None else bound + at_most)

    def set_host_length(self, tokens: int | None) -> None:
        """Tell the host side how many tokens every sequence holds (None: not known)
        after a captured graph has advanced the lengths on the device.  From here on the cache
        counts along again and reads nothing back: call it after the last replay."""
        self._captured = False
        self._note(tokens, tokens)

    def reset(self) -> None:
        """Forget every token (the memory is kept and written over)."""
        with self._on_device():
            self._lengths.zero_()
        if self._capturing():
            self._captured = True
        else:
            self._note(0, 0)


__all__ = ["QuantizedKVCache", "quantize_groups", "GROUP", "PAGE", "RANGE"]
