"""Logits before a token is drawn (sf_process_logits): penalties for repeated tokens, a bias, a mask of the tokens that
may follow.  No counterpart in the reference, which scores text and does not shape what a model answers.

For token t of a row, in float32 and in this order, rounded once to the logits' type:

    t occurs c > 0 times in the row's history:  x = x / repetition if x > 0 else x * repetition
                                                x = x - frequency * c;  x = x - presence
    x = x + bias[t]
    x = -inf if t is not allowed

One history serves all three penalties.  Where presence and frequency are to count the answer alone and repetition the
prompt too, two calls in float32 are the definition: one with the whole history and repetition, one of its result with
the answer and the rest.

A row whose mask allows nothing is -inf throughout.  Forward only: the result takes no gradient.

sample_logits draws the token (sf_sample_logits): temperature, top-k, top-p and min-p, with random numbers that the caller
gives.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L
from . import profiling as _prof
from .kernels import _written


def process_logits(logits: torch.Tensor, history: torch.Tensor | None = None,
                   history_lengths: torch.Tensor | None = None, *, repetition=1.0, presence=0.0, frequency=0.0,
                   bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """logits [B, V] (bf16 or float32, rows contiguous, e.g. all_logits[:, -1]) -> the processed logits, in `out` if
    given (logits itself may be given, or memory that overlaps it), else in a new tensor.

    history: int32 / int64 [B, n] token ids, the first history_lengths[b] (int32 [B], all where None) of a row counted;
    ids outside 0 .. V - 1 (padding) are not.  repetition, presence, frequency: a number, or float32 [B] on the device.
    bias: float32 [V] or [B, V].  allowed: bool [V] or [B, V], or its bits as int32 [ceil(V / 32)] or [B, ceil(V / 32)]
    (token t is bit t % 32 of word t // 32)."""
    dev = logits.device
    for t in (logits, history, history_lengths, bias, allowed, out):
        if t is not None and (not t.is_cuda or t.get_device() != dev.index):
            L.require_device_only(logits, history, history_lengths, bias, allowed, out)  # says which
    dt = L.dtype_code(logits)
    if logits.dim() != 2:
        raise ValueError(f"process_logits: logits must be [B, V], got {tuple(logits.shape)}")
    B, V = logits.shape
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    given = out
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    elif out.shape != (B, V) or out.dtype != logits.dtype or not (out.stride(1) == 1 or V <= 1) \
            or (B > 1 and out.stride(0) < V):
        raise ValueError(f"process_logits: out must be {logits.dtype} [{B}, {V}] with rows of its own")
    elif out.requires_grad and torch.is_grad_enabled():
        raise ValueError("process_logits: out requires grad, and what is written to it takes none")
    elif _mixed(logits, out):
        logits = logits.clone()
    n = 0
    if history is not None:
        if history.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"process_logits: the history is {history.dtype} (int32 / int64 only)")
        if history.dim() != 2 or history.shape[0] != B:
            raise ValueError(f"process_logits: history {tuple(history.shape)} for {B} rows")
        history = _rows(history)
        n = history.shape[1]
        if history_lengths is not None and (history_lengths.dtype != torch.int32 or history_lengths.shape != (B,)):
            raise ValueError(f"process_logits: history_lengths must be int32 [{B}]")
    elif history_lengths is not None:
        raise ValueError("process_logits: history_lengths without a history")
    rep, pres, freq = (_per_row(repetition, "repetition", B, dev), _per_row(presence, "presence", B, dev),
                       _per_row(frequency, "frequency", B, dev))
    if not isinstance(repetition, torch.Tensor) and not repetition > 0:
        raise ValueError(f"process_logits: a repetition penalty of {repetition}")
    if bias is not None:
        if bias.dtype != torch.float32:
            raise TypeError(f"process_logits: the bias is {bias.dtype} (float32 only)")
        if bias.shape not in ((V,), (B, V)):
            raise ValueError(f"process_logits: bias {tuple(bias.shape)} for logits {(B, V)}")
        bias = _rows(bias)
    bits = 0
    if allowed is not None:
        if allowed.dtype not in (torch.bool, torch.int32):
            raise TypeError(f"process_logits: allowed is {allowed.dtype} (bool, or int32 words of bits)")
        bits = int(allowed.dtype == torch.int32)
        wide = -(-V // 32) if bits else V
        if allowed.shape not in ((wide,), (B, wide)):
            raise ValueError(f"process_logits: allowed {tuple(allowed.shape)} for logits {(B, V)}")
        allowed = _rows(allowed)
    lengths = history_lengths.contiguous() if history_lengths is not None else None
    hist = (history.data_ptr(), history.stride(0), n, L.ptr(lengths) or 0) if n else (0, 0, 0, 0)
    desc = L.LOGITS_DESC.pack(
        logits.data_ptr(), out.data_ptr(), logits.stride(0) if B > 1 else V, out.stride(0) if B > 1 else V, B, V, *hist,
        rep[0], pres[0], freq[0], *_strided(bias), *_strided(allowed), rep[1], pres[1], freq[1],
        history.element_size() if n else 0, bits, dt)
    with _prof.region("sf_process_logits", 2 * B * V * logits.element_size(), "B", dev):
        L.check(L.lib().sf_process_logits(desc, L.stream(dev)), "sf_process_logits")
    _written(given)
    return out


def sample_logits(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  logprobs: bool = False):
    """A token for every row of logits [B, V] (bf16 or float32, any row stride, e.g. 0 for several draws from one row),
    drawn with uniform float32 [B] in [0, 1): ids int64 [B], or with logprobs (ids, float32 [B]).

    With w = exp((x - max x) / temperature), in the order of falling logit, equal ones by rising id, these are kept: the
    first top_k (0: all); of them the fewest first that hold top_p of their weight, and always the first; of them the ones
    with w >= min_p.  The token is the first, by id, at which the weight of the kept ones up to it exceeds uniform times
    their whole weight, its log-probability the logarithm of its share.  Temperature 0 takes the largest logit of the
    lowest id.  Each setting is a number, or a tensor [B] on the device (top_k int32, the others float32; what lies
    outside a setting's range there counts as its nearest end).  A row that holds a NaN, or nothing above -inf (a mask that
    allows nothing), has no token: -1, with a log-probability of NaN or -inf.  V is at most 262144.  Weights are whole
    numbers of 2^-44 of the largest (2^-43, 2^-42 above 65536, 131072 tokens), and a min_p above 0 keeps what has one of at
    least 1.  Forward only: the log-probabilities take no gradient."""
    dev = logits.device
    for t in (logits, uniform):
        if not t.is_cuda or t.get_device() != dev.index:
            L.require_device_only(logits, uniform)  # says which
    dt = L.dtype_code(logits)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"sample_logits: logits must be [B, V], got {tuple(logits.shape)}")
    B, V = logits.shape
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    if uniform.dtype != torch.float32 or uniform.shape != (B,):
        raise ValueError(f"sample_logits: uniform must be float32 [{B}], got {uniform.dtype} {tuple(uniform.shape)}")
    uniform = uniform.contiguous()
    temp, p, least = (_setting(x, name, low, high, B, dev) for x, name, low, high in
                      ((temperature, "temperature", 0.0, math.inf), (top_p, "top_p", 0.0, 1.0),
                       (min_p, "min_p", 0.0, 1.0)))
    k = _setting(top_k, "top_k", 0, 2 ** 31 - 1, B, dev, torch.int32)
    ids = torch.empty(B, dtype=torch.int64, device=dev)
    logp = torch.empty(B, dtype=torch.float32, device=dev) if logprobs else None
    desc = L.SAMPLE_DESC.pack(logits.data_ptr(), logits.stride(0) if B > 1 else V, B, V, uniform.data_ptr(),
                              ids.data_ptr(), L.ptr(logp) or 0, temp[0], k[0], p[0], least[0], temp[1], p[1], least[1],
                              k[1], dt)
    with L.on(dev), _prof.region("sf_sample_logits", B * V * logits.element_size(), "B", dev):
        L.check(L.lib().sf_sample_logits(desc, L.stream(dev)), "sf_sample_logits")
    return (ids, logp) if logprobs else ids


def _setting(x, name: str, low, high, B: int, dev, dtype=torch.float32) -> tuple:
    """A setting as the kernel takes it: a pointer to one for each row, or a number."""
    if not isinstance(x, torch.Tensor):
        if not low <= x <= high or (dtype == torch.int32 and int(x) != x):
            raise ValueError(f"sample_logits: a {name} of {x}")
        return 0, int(x) if dtype == torch.int32 else float(x)
    if x.device != dev:
        L.require_device_only(x)
        raise ValueError(f"sample_logits: {name} is on {x.device}, the logits on {dev}")
    if x.dtype != dtype or x.shape != (B,) or not x.is_contiguous():
        raise ValueError(f"sample_logits: {name} must be a number or a contiguous {dtype} [{B}]")
    return x.data_ptr(), 0


def _mixed(x: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether some row of out lies over another place of x's rows: it could be written before that is read."""
    B, V = x.shape
    by, start, end = x.element_size(), x.data_ptr(), out.data_ptr()
    xs, os = (t.stride(0) if B > 1 else V for t in (x, out))
    if start + by * (xs * (B - 1) + V) <= end or end + by * (os * (B - 1) + V) <= start:
        return False
    if xs != os or (end - start) % by:
        return True
    off = (end - start) // by
    return off != 0 and not V <= off % xs <= xs - V


def _strided(t: torch.Tensor | None) -> tuple[int, int]:
    """Address and row stride (0: one row for all); the bias' in elements, the mask's in bytes."""
    if t is None:
        return 0, 0
    step = t.stride(0) if t.dim() == 2 else 0
    return t.data_ptr(), step * (1 if t.dtype == torch.float32 else t.element_size())


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous rows (any row stride that goes forward)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _per_row(x, name: str, B: int, dev) -> tuple:
    """A penalty as the kernel takes it: a pointer to one for each row, or a number."""
    if not isinstance(x, torch.Tensor):
        return 0, float(x)
    if x.device != dev:
        L.require_device_only(x)
        raise ValueError(f"process_logits: {name} is on {x.device}, the logits on {dev}")
    if x.dtype != torch.float32 or x.shape != (B,) or not (x.is_contiguous()):
        raise ValueError(f"process_logits: {name} must be a number or a contiguous float32 [{B}]")
    return x.data_ptr(), 0.0
