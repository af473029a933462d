"""Distillation KL of Distill_Model (legacy/sparse_modeling.py:1749-1828) on the HIP kernels.

KL(P_teacher || Q_student) at temperature T over the vocabulary, logits
clamped to +-100; per chunk of token rows (sf_kl_chunk_rows: 2048, 512 or 128
by vocabulary size) a chunk with a NaN log-probability is skipped and a
non-finite chunk sum dropped; the total is scaled by T^2 / tokens and cast to
the student dtype (0 if not finite).  One fused pass reads both logit rows
(sf_kl_forward); the backward re-reads them (sf_kl_backward) and gives the
student gradient g (T / tokens) (q - p) inside the clamp range.  The teacher
takes no gradient (the reference computes it under no_grad).

Difference from the reference: for float32 logits the reference's
`.float().clamp_().mul_()` rewrites the caller's tensors in place; here the
inputs are left unchanged (the loss is the same).

Without the whole teacher (no counterpart in the reference): top_logits keeps the k largest logits of a teacher's rows
with the rows' log-sum-exp (sf_top_logits), and top_kl_loss is a student's KL from such a record (sf_top_kl_*).  For a row
with listed ids i_k and teacher logits t_k, at temperature T:

    a = s / T,   q = softmax(a) over the vocabulary,   p_k = exp(t_k / T - N)
    N = the teacher's log-sum-exp where the record holds it, and r = 1 - sum p is the probability of all other tokens;
        else log sum_k exp(t_k / T), and r = 0
    KL = sum_k p_k (log p_k - log q_(i_k)) + r (log r - log sum_(j unlisted) q_j)

and the loss T^2 sum w KL / sum w over the rows.  It can be differentiated twice (the Hutchinson probe does).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import profiling as _prof
from .linear import apply_in_backward, transforms_active


class _KL(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s2: torch.Tensor, t2: torch.Tensor, temperature: float, out_dtype: torch.dtype):
        dev = L.require_device(s2, t2)
        rows, vocab = s2.shape
        out = torch.empty((), dtype=out_dtype, device=dev)
        lse = torch.empty(rows, 2, dtype=torch.float64, device=dev)
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
        lib = L.lib()
        ws = torch.empty(max(int(lib.sf_kl_workspace_size(rows)), 1), dtype=torch.uint8, device=dev)
        with _prof.region("sf_kl_forward", 2 * s2.numel() * s2.element_size(), "B", dev):
            L.check(lib.sf_kl_forward(L.ptr(s2), L.ptr(t2), L.dtype_code(s2), rows, vocab, float(temperature),
                                      int(lib.sf_kl_chunk_rows(vocab)), L.ptr(out), L.dtype_code(out), L.ptr(lse),
                                      L.ptr(scale), L.ptr(ws), ws.numel(), L.stream(dev)), "sf_kl_forward")
        ctx.save_for_backward(s2, t2, lse, scale)
        ctx.temperature = float(temperature)
        return out

    @staticmethod
    def backward(ctx, g):
        s2, t2, lse, scale = ctx.saved_tensors
        # a Function of its own, so that torch.autograd.grad(..., create_graph=True) (the Hutchinson
        # Hessian-vector product) differentiates the KL gradient as the reference's torch ops are
        gs = apply_in_backward(_KLGrad, s2, t2, lse, scale, g, ctx.temperature)
        return gs, None, None, None


class _KLGrad(torch.autograd.Function):
    """gs = g * c_r * (q - p) inside the clamp range (sf_kl_backward), differentiable once more.

    With q = softmax(clamp(s) / T) per row, m = [-100 <= s <= 100] and c_r the row scale
    (T / rows, or 0 for a skipped chunk): d gs_i / d s_j = m_i m_j (g c_r / T) q_i (delta_ij - q_j),
    so the vector-Jacobian product with u = ggs * m is
        s_bar_j = m_j (g c_r / T) q_j (u_j - sum_i u_i q_i),
    and d gs / d g = c_r m (q - p) gives g_bar = sum ggs * c_r * m * (q - p).  These run as float32
    device elementwise ops and row sums (they are needed once per Hutchinson probe).  Rows of a dropped
    chunk (c_r = 0) give exact zeros even where their logits are NaN."""

    @staticmethod
    def forward(ctx, s2, t2, lse, scale, g, temperature: float):
        dev = s2.device
        gg = g.detach().contiguous()
        if gg.dtype not in (torch.float32, torch.bfloat16):
            gg = gg.float()
        gs = torch.empty_like(s2)
        rows, vocab = s2.shape
        with _prof.region("sf_kl_backward", 3 * s2.numel() * s2.element_size(), "B", dev):
            L.check(L.lib().sf_kl_backward(L.ptr(s2), L.ptr(t2), L.dtype_code(s2), rows, vocab, float(temperature),
                                           L.ptr(lse), L.ptr(scale), L.ptr(gg), L.dtype_code(gg), L.ptr(gs),
                                           L.stream(dev)), "sf_kl_backward")
        ctx.save_for_backward(s2, t2, lse, scale, g)
        ctx.temperature = float(temperature)
        return gs

    @staticmethod
    def backward(ctx, ggs):
        s2, t2, lse, scale, g = ctx.saved_tensors
        T = ctx.temperature
        s = s2.float()
        # live: inside the clamp range in a chunk the forward kept (row scale > 0).  A dropped chunk may hold
        # NaN logits (that is why it was dropped), and the reference takes it out of the graph, so every
        # term there is selected to 0 rather than multiplied by 0 (0 * NaN would be NaN).
        live = (s >= -100.0) & (s <= 100.0) & (scale > 0)[:, None]
        q = torch.where(live, torch.exp(s.clamp(-100.0, 100.0) / T - lse[:, 0:1].float()), 0.0)
        u = torch.where(live, ggs.float(), 0.0)
        dot = (u * q).sum(dim=1, keepdim=True)
        coef = (g.float() * scale / T)[:, None]
        s_bar = torch.where(live, coef * q * (u - dot), 0.0).to(s2.dtype)
        g_bar = None
        if ctx.needs_input_grad[4]:
            p = torch.where(live, torch.exp(t2.float().clamp(-100.0, 100.0) / T - lse[:, 1:2].float()), 0.0)
            g_bar = (u * (q - p) * scale[:, None]).sum().to(g.dtype).reshape(g.shape)
        return s_bar, None, None, None, g_bar, None


def chunked_kl_loss(student_logits: torch.Tensor, teacher_logits: torch.Tensor, temperature=2) -> torch.Tensor:
    """Distill_Model.kl_loss(student_logits, teacher_logits, temperature) (:1749-1828)."""
    shape = student_logits.shape
    dtype = student_logits.dtype
    s2 = student_logits.reshape(-1, shape[-1])
    t2 = teacher_logits.reshape(-1, shape[-1]).detach()
    if t2.dtype != s2.dtype:
        t2 = t2.to(s2.dtype)
    if s2.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"kl_loss: logits dtype {s2.dtype} (float32 / bfloat16 only)")
    return _KL.apply(s2.contiguous(), t2.contiguous(), float(temperature), dtype)


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
    at = state.data_ptr()  # the norm, then the rows' sums
    return L.TOP_KL_DESC.pack(s.data_ptr(), outer, step, inner, rows, s.shape[-1], values.data_ptr(), ids.data_ptr(),
                              values.shape[-1], L.ptr(lse) or 0, L.ptr(weights) or 0, at + 8, at, temperature,
                              L.dtype_code(s), L.dtype_code(values), ids.element_size()), s


def _top_kl_forward(s, values, ids, lse, weights, temperature: float):
    dev, lib, rows = s.device, L.lib(), s.shape[:-1].numel()
    loss = torch.empty((), dtype=torch.float32, device=dev)
    state = torch.empty(1 + int(lib.sf_top_kl_stats_size(rows)) // 8, dtype=torch.float64, device=dev)
    ws = torch.empty(int(lib.sf_top_kl_workspace_size(rows)), dtype=torch.uint8, device=dev)
    desc, keep = _top_kl_desc(s, values, ids, lse, weights, state, temperature)
    with L.on(dev), _prof.region("sf_top_kl_forward", s.numel() * s.element_size(), "B", dev):
        L.check(lib.sf_top_kl_forward(desc, loss.data_ptr(), ws.data_ptr(), ws.numel(), L.stream(dev)),
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
        dev, lib, u = s.device, L.lib(), u.contiguous()
        hs = torch.empty_like(s, memory_format=torch.contiguous_format)
        dot = torch.empty((), dtype=torch.float32, device=dev) if ctx.needs_input_grad[6] else None
        ws = torch.empty(int(lib.sf_top_kl_workspace_size(s.shape[:-1].numel())), dtype=torch.uint8, device=dev)
        desc, keep = _top_kl_desc(s, values, ids, lse, weights, state, ctx.temperature)
        with L.on(dev), _prof.region("sf_top_kl_double_backward", 3 * s.numel() * s.element_size(), "B", dev):
            L.check(lib.sf_top_kl_double_backward(desc, g.data_ptr(), u.data_ptr(), hs.data_ptr(), L.ptr(dot),
                                                  ws.data_ptr(), ws.numel(), L.stream(dev)),
                    "sf_top_kl_double_backward")
        return hs, None, None, None, None, None, dot, None


def top_kl_loss(student_logits: torch.Tensor, teacher: TopLogits, temperature=2, *,
                weights: torch.Tensor | None = None) -> torch.Tensor:
    """KL of a student's logits [.., V] (bf16 or float32, any strides with contiguous rows) from a teacher's top logits of
    the same rows, as float32 (see the module).

    weights: float32 [..], 1 where None; rows of weight 0 (prompts, padding) are not looked at and take a zero gradient.
    Rows without entries add 0; without any weight the loss is 0.  An id that is listed twice counts twice.  Logits are
    not clamped and nothing is dropped: what is not finite shows in the loss.  Only the student takes a gradient."""
    values, ids, lse, at = teacher
    dev = L.require_device_only(student_logits, values, ids, lse, weights)
    L.dtype_code(student_logits)
    L.dtype_code(values)
    lead, V = student_logits.shape[:-1], student_logits.shape[-1]
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
