"""Stateless ops: losses and activations (reference functional.py:8-89).

On CUDA tensors each op runs this package's kernels (fused softmax
cross-entropy, tanh-GELU, row softmax); on CPU they run PyTorch in float64,
matching the reference's Python-float semantics.
"""

from __future__ import annotations

import math

import torch

from underhfs_b200.tensor import Tensor


def _cuda_native(t: Tensor) -> bool:
    return t.device.kind == "cuda"


def mse_loss(input: Tensor, target: Tensor, reduction: str = "mean") -> Tensor:
    diff = input - target
    loss = diff * diff
    if reduction == "mean":
        return loss.mean()
    if reduction == "sum":
        return loss.sum()
    if reduction == "none":
        return loss
    raise ValueError(f"unsupported reduction: {reduction}")


def cross_entropy(logits: Tensor, target: Tensor, reduction: str = "mean") -> Tensor:
    """Mean/sum/none negative log-likelihood of integer targets.

    logits [batch, classes] (or [..., classes], flattened), target [batch].
    Matches the reference's clamp -log(max(p, 1e-30)).
    """
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unsupported reduction: {reduction}")
    if logits.ndim < 2:
        raise ValueError("cross_entropy expects logits with shape [batch, classes]")
    x = logits._data.reshape(-1, logits.shape[-1])
    tg = target._data.reshape(-1)
    if tg.shape[0] != x.shape[0]:
        raise ValueError(f"target batch {tg.shape[0]} does not match logits batch {x.shape[0]}")
    classes = x.shape[1]
    tgi = tg.to(torch.int64)
    bad = (tgi < 0) | (tgi >= classes)
    if bool(bad.any()):
        label = int(tgi[bad][0].item())
        raise ValueError(f"target class {label} is outside [0, {classes})")
    if _cuda_native(logits):
        from underhfs_b200.ops import functions as OF

        out = OF.cross_entropy(x, tgi, reduction)
        return Tensor._wrap(out, like=logits, backend="native_cuda")
    logp = torch.log_softmax(x, dim=-1)
    nll = -logp.gather(1, tgi.unsqueeze(1)).squeeze(1)
    nll = torch.clamp(nll, max=-math.log(1e-30))
    if reduction == "mean":
        nll = nll.sum() / max(1, x.shape[0])
    elif reduction == "sum":
        nll = nll.sum()
    return Tensor._wrap(nll, like=logits)


def relu(input: Tensor) -> Tensor:
    return input.relu()


def gelu(input: Tensor) -> Tensor:
    """tanh-approximation GELU: 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3)))."""
    if _cuda_native(input):
        from underhfs_b200.ops import functions as OF

        return Tensor._wrap(OF.gelu(input._data), like=input, backend="native_cuda")
    x = input._data
    c = math.sqrt(2.0 / math.pi)
    return Tensor._wrap(0.5 * x * (1.0 + torch.tanh(c * (x + 0.044715 * x * x * x))), like=input)


def softmax(input: Tensor) -> Tensor:
    return input.softmax()


_SETTINGS = {"temperature": (0.0, 1e30), "top_k": (0, 2**31 - 1), "top_p": (0.0, 1.0), "min_p": (0.0, 1.0)}


def check_sampling(**settings) -> None:
    """Raise ValueError for a sampling setting, given as a number, that ``sample`` would refuse."""
    for name, value in settings.items():
        low, high = _SETTINGS[name]
        if not isinstance(value, (torch.Tensor, Tensor)) and not low <= value <= high:  # False for NaN
            raise ValueError(f"{name} must lie in [{low:g}, {high:g}], got {value}")


def _setting(value, name: str, rows: int, device: torch.device, dtype: torch.dtype):
    """A sampling setting: a checked number, or a tensor with one value per row."""
    if not isinstance(value, (int, float)):
        value = value._data if isinstance(value, Tensor) else value
    if isinstance(value, torch.Tensor):
        if value.numel() != rows:
            raise ValueError(f"{name} needs one value for each of {rows} rows, got {list(value.shape)}")
        if value.device != device:
            raise RuntimeError(f"{name} is on {value.device}, the logits on {device}")
        if value.dtype == dtype and value.dim() == 1 and value.is_contiguous():
            return value
        value = value.detach().reshape(-1)
        if dtype == torch.int32 and value.dtype == torch.int64:
            value = value.clamp(0, 2**31 - 1)  # <= 0 is off
        return value.to(dtype).contiguous()
    low, high = _SETTINGS[name]
    if not low <= value <= high:
        check_sampling(**{name: value})
    return int(value) if dtype == torch.int32 else float(value)


def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> Tensor:
    """The next token of each row of logits [..., vocab], chosen by ``uniform``
    [...] (numbers in [0, 1)); int64 [...].

    In this order: ``top_k`` > 0 keeps the k largest logits; ``top_p`` < 1 keeps,
    of those, the fewest largest whose probabilities reach top_p; ``min_p`` keeps
    tokens of at least min_p times the largest probability.  Equal logits are
    taken by lowest index.  Probabilities are softmax(logits / temperature); the
    token is the first, by index, at which the running sum of the kept ones
    passes uniform times their sum.  ``temperature`` 0 takes the largest logit
    (lowest index).  Each setting is a number or a tensor with one value per
    row (a temperature <= 0, a top_k <= 0 and a top_p >= 1 there are "off"; at
    least the largest logit is always kept).

    Logits of -inf and NaN are never chosen; a row without any other gives -1.
    On CUDA (fp32, fp16, bf16, vocabularies up to 327680) this is one kernel
    whose result does not depend on how the row is split; on the CPU it runs in
    float64.  No gradient flows through the choice.
    """
    x = logits._data if isinstance(logits, Tensor) else logits
    u = uniform._data if isinstance(uniform, Tensor) else uniform
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"sample expects logits [..., vocab], got {list(x.shape)}")
    if not x.is_floating_point():
        raise TypeError(f"logits must be floating-point, got {x.dtype}")
    if u.shape != x.shape[:-1]:
        raise ValueError(f"uniform must have shape {list(x.shape[:-1])}, got {list(u.shape)}")
    if u.device != x.device:
        raise RuntimeError(f"uniform is on {u.device}, the logits on {x.device}")
    shape, vocab = x.shape[:-1], x.shape[-1]
    if x.dim() != 2:
        x = x.detach().reshape(-1, vocab)
    rows = x.shape[0]
    real = torch.float32 if x.is_cuda else torch.float64
    if u.dim() != 1 or u.dtype != real or not u.is_contiguous():
        u = u.detach().reshape(-1).to(real).contiguous()
    temperature = _setting(temperature, "temperature", rows, x.device, real)
    top_k = _setting(top_k, "top_k", rows, x.device, torch.int32)
    top_p = _setting(top_p, "top_p", rows, x.device, real)
    min_p = _setting(min_p, "min_p", rows, x.device, real)
    if x.is_cuda:
        from underhfs_b200.ops import kernels as K

        if vocab > 327680:
            raise ValueError(f"the CUDA kernel takes vocabularies up to 327680, got {vocab}")
        if x.device.index == torch._C._cuda_getDevice():
            token = K.sample_tokens(x, u, temperature, top_k, top_p, min_p)
        else:
            with torch.cuda.device(x.device):
                token = K.sample_tokens(x, u, temperature, top_k, top_p, min_p)
    else:
        token = _sample_cpu(x.detach().double(), u.detach(), temperature, top_k, top_p, min_p)
    return Tensor._wrap(token if len(shape) == 1 else token.reshape(shape))


def _sample_cpu(x: torch.Tensor, u: torch.Tensor, temperature, top_k, top_p, min_p) -> torch.Tensor:
    rows, vocab = x.shape

    def column(v):
        v = v.double() if isinstance(v, torch.Tensor) else torch.full((rows,), float(v), dtype=torch.float64)
        return v.reshape(-1, 1)

    temperature, top_k, top_p, min_p = (column(v) for v in (temperature, top_k, top_p, min_p))
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    top = val[:, :1]
    t = torch.where(temperature > 0, temperature, torch.ones_like(temperature)).clamp(1e-30, 1e30)
    # the largest logit's own weight is 1, infinite or not
    w = torch.where(val == top, torch.ones_like(val), torch.exp((val - top) / t)) * (val > -math.inf)
    rank = torch.arange(vocab).unsqueeze(0)
    w = w * ((top_k <= 0) | (rank < top_k))
    before = torch.cumsum(w, 1) - w
    keep = ~(top_p < 1.0) | (before < top_p * w.sum(1, keepdim=True)) | (rank == 0)
    w = w * keep * ((w >= min_p) | (val == top))
    run = torch.cumsum(torch.zeros_like(w).scatter_(1, idx, w), 1)
    total = run[:, -1:]
    goal = torch.nan_to_num(u.reshape(-1, 1), nan=0.0).clamp(0.0, 1.0) * total
    last = (run < total).sum(1)  # the last kept token, where a goal of the whole sum ends
    token = torch.minimum((run <= goal).sum(1), last)
    token = torch.where(temperature[:, 0] > 0, token, idx[:, 0])
    return torch.where(top[:, 0] > -math.inf, token, torch.full_like(token, -1))
