"""Rotary positions for queries and keys (sf_rotary): half or interleaved pairs, the whole head or part of it, one
position for each token, tables scaled for contexts longer than the trained one.

Pair i of a head, at position p, turns by the angle p f_i:

    a' = a c - b s,  b' = b c + a s,   c = m cos(p f_i),  s = m sin(p f_i),   f_i = theta^(-2 i / rotary_dim)

Scalings for a context `factor` times the trained one:

    linear  f_i / factor: positions interpolated (Chen et al., 2023)
    ntk     theta factor^(r / (r - 2)) for theta, r = rotary_dim: the slowest pair interpolates, the fastest stays
    yarn    f_i (g + (1 - g) / factor), g = clamp((L f_i / 2 pi - beta_slow) / (beta_fast - beta_slow), 0, 1), L the
            trained context: pairs that turn often within it stay, those that turn less than once interpolate;
            m = 0.1 ln(factor) + 1 (Peng et al., 2023).  m is 1 otherwise.  The ramp g is linear in a pair's turns, as
            in the paper; a model trained with one linear in the pair's index i has other frequencies inside the ramp
            and needs tables made for it, which rotary_embed takes like these.

There is no counterpart in the reference, whose attention rotates whole heads by the positions 0 .. S - 1 in half
pairs (HuggingFace's eager attention, legacy/model_llama.py:39-55; llama.causal_attention does that).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib as L
from . import profiling as _prof
from .linear import plain_backward, transforms_active

SCALINGS = ("linear", "ntk", "yarn")


@dataclass(frozen=True)
class RotaryScaling:
    """How the angles change for a context `factor` times the trained one (see the module)."""

    kind: str
    factor: float
    original_length: int = 0  # yarn: the trained context
    beta_fast: float = 32.0   # yarn: turns within it from which a pair stays as it is
    beta_slow: float = 1.0    # yarn: turns up to which a pair interpolates

    def __post_init__(self):
        if self.kind not in SCALINGS:
            raise ValueError(f"RotaryScaling: kind {self.kind!r} is none of {SCALINGS}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"RotaryScaling: factor {self.factor} must be finite and at least 1")
        if self.kind == "yarn" and self.original_length < 1:
            raise ValueError("RotaryScaling: yarn needs the original_length that the model was trained on")
        if not self.beta_fast > self.beta_slow:
            raise ValueError("RotaryScaling: beta_fast must exceed beta_slow")


def rotary_cos_sin(positions: int, rotary_dim: int, theta: float = 10000.0, scaling: RotaryScaling | None = None,
                   device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos, sin [positions, rotary_dim / 2] in float32 of positions 0 .. positions - 1, for rotary_embed.  The angles
    are taken in float64 (an angle in float32 is off by 2^-24 of itself: 0.004 of a turn's radian at 65536)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_cos_sin: rotary_dim {rotary_dim} must be even and at least 2")
    if positions < 1:
        raise ValueError(f"rotary_cos_sin: {positions} positions")
    m = 1.0
    if scaling is not None and scaling.kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("rotary_cos_sin: ntk scaling needs a rotary_dim of 4 or more")
        theta = theta * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / -rotary_dim)
    if scaling is not None and scaling.kind == "linear":
        f = f / scaling.factor
    elif scaling is not None and scaling.kind == "yarn":
        turns = scaling.original_length * f / (2.0 * math.pi)
        g = ((turns - scaling.beta_slow) / (scaling.beta_fast - scaling.beta_slow)).clamp_(0.0, 1.0)
        f = f * (g + (1.0 - g) / scaling.factor)
        m = 0.1 * math.log(scaling.factor) + 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f[None]
    return (m * angle.cos()).float(), (m * angle.sin()).float()


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor | None = None, interleaved: bool = False):
    """q [B, S, H, D] and k [B, S, Hk, D] (or None) turned by their positions -> (q', k'), contiguous, in one launch.

    cos, sin: float32 [P, r / 2] (rotary_cos_sin); the first r elements of a head turn, the others are copied.
    positions: int32 or int64 [B, S] or [S] on the device, None for 0 .. S - 1; one outside 0 .. P - 1 gives NaN.
    q and k are bf16 or float32 and may be views (columns of a fused projection); the turn is in float32, rounded
    once.  Differentiable in q and k any number of times, in reverse mode (forward mode raises); the tables and positions
    take no gradient."""
    _check(q, k, cos, sin, positions)
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) or transforms_active():
        return _Rotary.apply(q, k, cos, sin, positions, bool(interleaved), False)
    return _launch(q, k, cos, sin, positions, interleaved, False)


def _check(q, k, cos, sin, positions) -> None:
    at = q.get_device()
    if at < 0 or cos.get_device() != at or sin.get_device() != at or (k is not None and k.get_device() != at) \
            or (positions is not None and positions.get_device() != at):
        L.require_device_only(q, k, cos, sin, positions)  # says which
    if q.dim() != 4:
        raise ValueError(f"rotary_embed: q must be [B, S, H, D], got {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"rotary_embed: q is {q.dtype} (bfloat16 / float32 only)")
    B, S, _, D = q.shape
    if k is not None:
        if k.dim() != 4 or k.shape[0] != B or k.shape[1] != S or k.shape[3] != D:
            raise ValueError(f"rotary_embed: k {tuple(k.shape)} does not go with q {tuple(q.shape)}")
        if k.dtype != q.dtype:
            raise TypeError(f"rotary_embed: k is {k.dtype}, q {q.dtype}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("rotary_embed: cos and sin must be float32")
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError(f"rotary_embed: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be [P, r / 2] both")
    if not 1 <= cos.shape[1] <= D // 2:
        raise ValueError(f"rotary_embed: tables of {cos.shape[1]} pairs for heads of {D}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("rotary_embed: cos and sin take no gradient")
    if positions is None:
        if S > cos.shape[0]:
            raise ValueError(f"rotary_embed: {S} positions, the tables hold {cos.shape[0]}")
    elif positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"rotary_embed: positions are {positions.dtype} (int32 / int64 only)")
    elif positions.shape != (B, S) and positions.shape != (S,):
        raise ValueError(f"rotary_embed: positions {tuple(positions.shape)} for q {tuple(q.shape)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous heads (any other strides)."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


_NONE = (0, 0, 0, 0, 0, 0)


def _side(t: torch.Tensor, y: torch.Tensor) -> tuple:
    sb, ss, sh, _ = t.stride()
    return t.data_ptr(), y.data_ptr(), sb, ss, sh, t.shape[2]


def _launch(q, k, cos, sin, positions, interleaved: bool, inverse: bool):
    some = q if q is not None else k
    B, S, _, D = some.shape
    cos, sin = cos.contiguous(), sin.contiguous()
    at = (0, 0, 0)
    if positions is not None:
        positions = positions.contiguous()
        at = positions.data_ptr(), S if positions.dim() == 2 else 0, positions.element_size()
    q_out = k_out = None
    q_side = k_side = _NONE
    if q is not None:
        q = _rows(q)
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q_side = _side(q, q_out)
    if k is not None:
        k = _rows(k)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        k_side = _side(k, k_out)
    desc = L.ROTARY_DESC.pack(*q_side, *k_side, B, S, D, 2 * cos.shape[1], cos.data_ptr(), sin.data_ptr(),
                              cos.shape[0], *at, L.dtype_code(some), interleaved, inverse)
    dev = some.device
    with _prof.region("sf_rotary", 2 * (q_side[5] + k_side[5]) * B * S * D * some.element_size(), "B", dev):
        L.check(L.lib().sf_rotary(desc, L.stream(dev)), "sf_rotary")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The turn, or with `inverse` its adjoint; the backward of each is the other."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved: bool, inverse: bool):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos, sin, positions)
        ctx.form = (interleaved, inverse)
        return _launch(q, k, cos, sin, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        interleaved, inverse = ctx.form
        # an output that no derivative reaches comes as None
        gq, gk = (g if n else None for g, n in zip((gq, gk), ctx.needs_input_grad))
        if gq is None and gk is None:
            return (None,) * 7
        turn = _launch if plain_backward() else _Rotary.apply
        return (*turn(gq, gk, cos, sin, positions, interleaved, not inverse), None, None, None, None, None)
