"""Distillation from a teacher's top logits (sf_top_logits, sf_top_kl_*; no counterpart in the reference, whose
Distill_Model.kl_loss takes every logit of a teacher that runs beside the student).

top_logits keeps the k largest logits of a teacher's rows with the rows' log-sum-exp, and top_kl_loss is a student's KL
from such a record.  For a row with listed ids i_k and teacher logits t_k, at temperature T:

    a = s / T,   q = softmax(a) over the vocabulary,   p_k = exp(t_k / T - N)
    N = the teacher's log-sum-exp where the record holds it, and r = 1 - sum p is the probability of all other tokens;
        else log sum_k exp(t_k / T), and r = 0
    KL = sum_k p_k (log p_k - log q_(i_k)) + r (log r - log sum_(j unlisted) q_j)

and the loss T^2 sum w KL / sum w over the rows.  It can be differentiated twice (the Hutchinson probe does).
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import profiling as _prof
from .linear import apply_in_backward, transforms_active


class TopLogits(NamedTuple):
    """The largest logits of rows [..], as top_logits gives them or as they were stored.

    values [.., k] (bfloat16 / float32), ids [.., k] (int32 / int64; those outside the vocabulary are padding), lse
    float32 [..]: log sum exp(logits / temperature) over the whole vocabulary, or None where only the listed tokens are
    to count; temperature: the one that lse was taken at."""

    values: torch.Tensor
    ids: torch.Tensor
    lse: torch.Tensor | None = None
    temperature: float | None = None


def top_logits(logits: torch.Tensor, k: int, temperature=2) -> TopLogits:
    """The k largest logits [.., V] of every row (bf16 or float32), falling, equal ones by rising id (NaN above all), with
    int32 ids and the row's log-sum-exp at the temperature.  k is at most 1024, V at most 262144.  values - lse at a
    temperature of 1 are the tokens' log-probabilities.  The result takes no gradient."""
    dev = L.require_device_only(logits)
    dt = L.dtype_code(logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"top_logits: logits must be [.., V], got {tuple(logits.shape)}")
    lead, V, k = logits.shape[:-1], logits.shape[-1], int(k)
    if not 1 <= k <= V:
        raise ValueError(f"top_logits: the {k} largest of {V}")
    temperature = float(temperature)
    if not temperature > 0.0:
        raise ValueError(f"top_logits: a temperature of {temperature}")
    logits, outer, step, inner, rows = L.rows_of(logits.detach())
    values = torch.empty(*lead, k, dtype=logits.dtype, device=dev)
    ids = torch.empty(*lead, k, dtype=torch.int32, device=dev)
    lse = torch.empty(lead, dtype=torch.float32, device=dev)
    desc = L.TOP_LOGITS_DESC.pack(logits.data_ptr(), outer, step, inner, rows, V, k, values.data_ptr(), ids.data_ptr(),
                                  lse.data_ptr(), temperature, dt)
    with L.on(dev), _prof.region("sf_top_logits", rows * V * logits.element_size(), "B", dev):
        L.check(L.lib().sf_top_logits(desc, L.stream(dev)), "sf_top_logits")
    return TopLogits(values, ids, lse, temperature)


def _top_kl_desc(s, values, ids, lse, weights, state, temperature):
    """The descriptor, and s or the copy of it that has to live until the call."""
    s, outer, step, inner, rows = L.rows_of(s)
    at = state.data_ptr()  # the norm, the rows' sums, the forward's workspace
    return L.TOP_KL_DESC.pack(s.data_ptr(), outer, step, inner, rows, s.shape[-1], values.data_ptr(), ids.data_ptr(),
                              values.shape[-1], L.ptr(lse) or 0, L.ptr(weights) or 0, at + 8, at, temperature,
                              L.dtype_code(s), L.dtype_code(values), ids.element_size()), s


@lru_cache(maxsize=64)
def _sizes(rows: int) -> tuple[int, int]:
    """Bytes of the rows' sums and of the workspace."""
    return int(L.lib().sf_top_kl_stats_size(rows)), int(L.lib().sf_top_kl_workspace_size(rows))


def _top_kl_forward(s, values, ids, lse, weights, temperature: float):
    dev, (stats, ws) = s.device, _sizes(s.shape[:-1].numel())
    loss = torch.empty((), dtype=torch.float32, device=dev)
    state = torch.empty(1 + (stats + ws) // 8, dtype=torch.float64, device=dev)  # an allocation costs 1.5 us
    desc, keep = _top_kl_desc(s, values, ids, lse, weights, state, temperature)
    with L.on(dev), _prof.region("sf_top_kl_forward", s.numel() * s.element_size(), "B", dev):
        L.check(L.lib().sf_top_kl_forward(desc, loss.data_ptr(), state.data_ptr() + 8 + stats, ws, L.stream(dev)),
                "sf_top_kl_forward")
    return loss, state


class _TopKL(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, values, ids, lse, weights, temperature: float):
        loss, state = _top_kl_forward(s, values, ids, lse, weights, temperature)
        ctx.save_for_backward(s, values, ids, lse, weights, state)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, g):
        # a Function of its own, as the whole KL's gradient: the Hutchinson probe differentiates it
        return apply_in_backward(_TopKLGrad, *ctx.saved_tensors, g, ctx.temperature), None, None, None, None, None


class _TopKLGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, values, ids, lse, weights, state, g, temperature: float):
        dev = s.device
        gs = torch.empty_like(s, memory_format=torch.contiguous_format)
        desc, keep = _top_kl_desc(s, values, ids, lse, weights, state, temperature)
        with L.on(dev), _prof.region("sf_top_kl_backward", 2 * s.numel() * s.element_size(), "B", dev):
            L.check(L.lib().sf_top_kl_backward(desc, g.data_ptr(), gs.data_ptr(), L.stream(dev)), "sf_top_kl_backward")
        ctx.save_for_backward(s, values, ids, lse, weights, state, g)
        ctx.temperature = temperature
        return gs

    @staticmethod
    @once_differentiable
    def backward(ctx, u):
        s, values, ids, lse, weights, state, g = ctx.saved_tensors
        dev, u = s.device, u.contiguous()
        hs = torch.empty_like(s, memory_format=torch.contiguous_format)
        dot = torch.empty((), dtype=torch.float32, device=dev) if ctx.needs_input_grad[6] else None
        ws = torch.empty(_sizes(s.shape[:-1].numel())[1], dtype=torch.uint8, device=dev)
        desc, keep = _top_kl_desc(s, values, ids, lse, weights, state, ctx.temperature)
        with L.on(dev), _prof.region("sf_top_kl_double_backward", 3 * s.numel() * s.element_size(), "B", dev):
            L.check(L.lib().sf_top_kl_double_backward(desc, g.data_ptr(), u.data_ptr(), hs.data_ptr(), L.ptr(dot),
                                                      ws.data_ptr(), ws.numel(), L.stream(dev)),
                    "sf_top_kl_double_backward")
        return hs, None, None, None, None, None, dot, None


def top_kl_loss(student_logits: torch.Tensor, teacher: TopLogits, temperature=2, *,
                weights: torch.Tensor | None = None) -> torch.Tensor:
    """KL of a student's logits [.., V] (bf16 or float32, any strides with contiguous rows) from a teacher's top logits of
    the same rows, as float32 (see the module).

    weights: float32 [..], 1 where None; rows of weight 0 (prompts, padding) are not looked at and take a zero gradient.
    Rows without entries, or without a log-sum-exp and with entries of -inf alone, add 0; without any weight the loss is 0.
    An id that is listed twice counts twice.  A row has at most 4096 entries, and no more than V.  Logits are not clamped
    and nothing is dropped: what is not finite shows in the loss, a log-sum-exp of -inf (a teacher's row that is masked
    throughout) too.  Only the student takes a gradient.  Temperatures lie in 1e-30 .. 1e30."""
    values, ids, lse, at = teacher
    dev = L.require_device_only(student_logits, values, ids, lse, weights)
    L.dtype_code(student_logits)
    L.dtype_code(values)
    if student_logits.dim() < 1:
        raise ValueError("top_kl_loss: the logits must be [.., V], got a number")
    lead = student_logits.shape[:-1]
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"top_kl_loss: the ids are {ids.dtype} (int32 / int64 only)")
    if values.shape != ids.shape or values.shape[:-1] != lead:
        raise ValueError(f"top_kl_loss: values {tuple(values.shape)}, ids {tuple(ids.shape)} for logits "
                         f"{tuple(student_logits.shape)}")
    temperature = float(temperature)
    if not temperature > 0.0:
        raise ValueError(f"top_kl_loss: a temperature of {temperature}")
    for name, t in (("lse", lse), ("weights", weights)):
        if t is not None and (t.dtype != torch.float32 or t.shape != lead):
            raise ValueError(f"top_kl_loss: {name} must be float32 {list(lead)}, got {t.dtype} {tuple(t.shape)}")
    if lse is not None and at is not None and float(at) != temperature:
        raise ValueError(f"top_kl_loss: the record's log-sum-exp is at temperature {at}, the loss at {temperature}")
    if lead.numel() == 0:
        return student_logits.sum(dtype=torch.float32)
    args = (student_logits, _given(values), _given(ids), _given(lse), _given(weights), temperature)
    if not (student_logits.requires_grad and torch.is_grad_enabled()) and not transforms_active():
        return _top_kl_forward(*args)[0]
    return _TopKL.apply(*args)


def _given(t: torch.Tensor | None) -> torch.Tensor | None:
    """An input that takes no gradient, contiguous."""
    if t is None:
        return None
    t = t.detach() if t.requires_grad else t
    return t if t.is_contiguous() else t.contiguous()
