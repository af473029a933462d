"""Drop-in SparseLinear / Distill_Model on the MI355X HIP kernels.

Mirrors the interface of liuhanzuo/SparseForge legacy/sparse_modeling.py:
the same class names, constructor signatures, parameter names (``mask``,
``grad_ema``, ``hessian_diag``, ``frozen_mask_flags``, ``scaler_row``,
``x_proj``, ``SLoRB_Weight``, the ``weight.mask`` alias), methods and
exceptions.  The tensor work runs in the sparseforge_amd HIP library:

* forward / backward of the masked linear: bf16 or f32 MFMA GEMMs, SLoRB
  folded into the same GEMMs.  A soft or mixed effective mask is applied by
  one elementwise pass that writes W * E for the forward GEMM (kept for the
  input-gradient GEMM); the double backward applies the mask inside the GEMM
  while W tiles are staged;
* compute_gate_target / update_mask: score statistics, tau quantile and one
  fused gate + penalty + EMA + freeze + flip-count pass over the layer;
* _hard_mask_from_soft: the N:M projection with torch.topk's tie order.

Everything runs on the GPU; CPU tensors raise (there is no CPU path).
"""
from __future__ import annotations

import math
import warnings
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
from torch.nn import functional as F

from . import _lib as L
from . import block_masks as BM
from . import kernels as K
from . import schedules as SCH


# FusedMaskedLinearSTE lives with the GEMM ops.
from .linear import FusedMaskedLinearSTE, masked_linear  # noqa: E402


SORTED_SAMPLE_MAX = 1 << 28  # sf_sample_indices_sorted's sample-size bound


def draw_samples(size: int, ns, seeds, device) -> torch.Tensor:
    """[len(ns), size] tau samples, row c uniform over [0, ns[c]) from seeds[c]: sorted draws from the
    library's sampler, or (samples of 2^28 and more) torch.randint from a generator seeded with seeds[c],
    unsorted, which the batched update gathers instead of folding."""
    if size < SORTED_SAMPLE_MAX:
        return K.sample_indices_sorted(size, ns, seeds, device)
    out = torch.empty((len(ns), size), dtype=torch.int64, device=device)
    for c, (n, seed) in enumerate(zip(ns, seeds)):
        gen = torch.Generator(device=device).manual_seed(int(seed))
        out[c] = torch.randint(0, int(n), (size,), generator=gen, device=device)
    return out


@dataclass
class SparseLinearConfig:
    """Mask knobs of a SparseLinear (legacy/sparse_modeling.py:136-239), same fields and defaults."""

    change_mask: bool = True
    mode: str = "sparse_forward"
    mask_type: str = "structured"
    mask_metric: str = "hessian_obd"
    sparsity_ratio: float = 0.5
    N: int = 2
    M: int = 4
    beta: float = 0.99
    score_ema_beta: float = 0.99
    mask_update_period: int = 10
    mask_update_switch_step: int = 0
    mask_update_period_before: Optional[int] = None
    mask_update_period_after: Optional[int] = None
    mask_lr: float = 0.10
    mask_penalty_lr: float = None
    mask_penalty_mode: str = "mid"
    temp_init: float = 1.0
    temp_min: float = 0.05
    temp_decay: float = 0.97
    mask_binarize_decay: float = 0
    mask_hardening_start: int = 1000
    mask_hardening_duration: int = 10000
    sparsity_warmup_steps: int = 100
    tau_sample_size: int = 262144
    temperature: float = 1.0
    freeze_low: float = 0.0
    freeze_high: float = 1.0
    SLoRB: bool = False
    SLoRB_k: int = 64
    SLoRB_init_type: str = "mean"
    trainable_projection: bool = False
    structured_exact: bool = False
    hard_mask_type: str = "match"
    beta_structural_start: int = 0
    beta_structural_end: int = 0
    gradient_checkpointing: bool = False
    srste_decay: float = 0.0
    glu_joint_mask: bool = False
    weight_scaling: bool = False


_BLOCK_TYPES = ("block16", "block_sparse16", "block_sparse32")


def _dtype_tag(dt: torch.dtype) -> int:
    if dt == torch.float32:
        return L.DT_F32
    if dt == torch.bfloat16:
        return L.DT_BF16
    raise TypeError(f"sparseforge_amd: unsupported dtype {dt}")


class SparseLinear(nn.Linear):
    """Continuous-mask pruning linear layer (legacy/sparse_modeling.py:242-1666) on HIP kernels."""

    def __init__(self, in_features, out_features, sparselinear_config=None, bias=True, **kwargs):
        super().__init__(in_features, out_features, bias=bias, **kwargs)
        assert sparselinear_config is not None
        cfg = sparselinear_config
        self.cfg = cfg
        self.mode = cfg.mode
        self.change_mask = cfg.change_mask
        self.mask_type = cfg.mask_type
        self.mask_metric = cfg.mask_metric
        self.sparsity_ratio = cfg.sparsity_ratio
        self.N = cfg.N
        self.M = cfg.M

        dev, dtype = self.weight.device, self.weight.dtype
        # State tensors are frozen Parameters in the weight dtype; a size-1
        # placeholder stands in when the config does not need one (:284-367).
        self.mask = nn.Parameter(torch.ones(out_features, in_features, device=dev, dtype=dtype), requires_grad=False)

        def _state(full: bool, name: str, shape):
            if full:
                return nn.Parameter(torch.zeros(*shape, device=dev, dtype=dtype), requires_grad=False)
            setattr(self, f"_{name}_placeholder", True)
            return nn.Parameter(torch.zeros(1, device=dev, dtype=dtype), requires_grad=False)

        self.grad_ema = _state(cfg.change_mask and cfg.mask_metric == "movement", "grad_ema",
                               (out_features, in_features))
        need_h = cfg.change_mask and (cfg.mask_metric in ("hessian_obd", "hessian_ratio", "hessian")
                                      or getattr(cfg, "enable_hutchinson", False))
        self.hessian_diag = _state(need_h, "hessian_diag", (out_features, in_features))
        need_frozen = cfg.change_mask and ((cfg.freeze_low > 0.0) or (cfg.freeze_high < 1.0))
        self.frozen_mask_flags = _state(need_frozen, "frozen_mask_flags", (out_features, in_features))
        self.scaler_row = _state(cfg.mask_metric == "wanda", "scaler_row", (in_features,))
        self.nsamples = 0

        self.weight.mask = self.mask
        self.weight.flipped_mask = 0
        self.weight.init_flipped_mask = 0
        self.weight.param_count = self.weight.numel()
        self.srste_decay = cfg.srste_decay
        self.mask_penalty_lr = (float(cfg.mask_penalty_lr) if getattr(cfg, "mask_penalty_lr", None) is not None
                                else float(cfg.mask_lr))
        self.hard_mask_type = str(getattr(cfg, "hard_mask_type", "match") or "match")
        self.hardening_x = 1.0

        self.SLoRB = cfg.SLoRB
        if self.SLoRB:
            self.SLoRB_k = cfg.SLoRB_k
            self.SLoRB_init_type = cfg.SLoRB_init_type
            self.trainable_projection = cfg.trainable_projection
            k = int(self.SLoRB_k)
            assert k > 0, f"SLoRB_k must be > 0 (got {k})"
            assert in_features % k == 0, f"in_features ({in_features}) must be divisible by SLoRB_k ({k})."
            rows = in_features // k
            self.x_proj = nn.Parameter(torch.zeros(rows, in_features, device=dev, dtype=dtype),
                                       requires_grad=bool(self.trainable_projection))
            self.SLoRB_Weight = nn.Parameter(torch.zeros(out_features, rows, device=dev, dtype=dtype),
                                             requires_grad=True)

    # ---- placeholders -----------------------------------------------------
    def _is_placeholder(self, name: str) -> bool:
        return getattr(self, f"_{name}_placeholder", False)

    # ---- init ---------------------------------------------------------------
    @torch.no_grad()
    def initialize(self):
        """(:410-439)"""
        self.mask.fill_(1.0)
        if not self._is_placeholder("frozen_mask_flags"):
            self.frozen_mask_flags.zero_()
        if not self._is_placeholder("grad_ema"):
            self.grad_ema.zero_()
        if not self._is_placeholder("hessian_diag"):
            if self.mask_metric == "hessian_obd":
                self.hessian_diag.fill_(1.0)
            else:
                self.hessian_diag.zero_()
        self.weight.mask = self.mask
        self.weight.flipped_mask = 0
        self.weight.init_flipped_mask = 0

    @torch.no_grad()
    def sync_weight(self):
        """(:441-458)"""
        self.weight.mask = self.mask
        try:
            self.weight.flipped_mask = int(getattr(self.weight, "flipped_mask", 0))
        except Exception:
            self.weight.flipped_mask = 0
        try:
            self.weight.init_flipped_mask = int(getattr(self.weight, "init_flipped_mask", 0))
        except Exception:
            self.weight.init_flipped_mask = 0
        try:
            self.weight.param_count = int(getattr(self.weight, "param_count", self.weight.numel()))
        except Exception:
            self.weight.param_count = self.weight.numel()

    @torch.no_grad()
    def init_SLoRB(self):
        """Block-sum projection and SLoRB weight init (:830-872)."""
        Nout, d = self.weight.shape
        k = int(self.SLoRB_k)
        assert d % k == 0, f"in_features ({d}) must be divisible by SLoRB_k ({k})."
        rows = d // k
        dev = self.weight.device
        if not hasattr(self, "x_proj") or not isinstance(self.x_proj, nn.Parameter):
            self.x_proj = nn.Parameter(torch.zeros(rows, d, device=dev, dtype=self.weight.dtype),
                                       requires_grad=bool(self.trainable_projection))
        if not hasattr(self, "SLoRB_Weight") or not isinstance(self.SLoRB_Weight, nn.Parameter):
            self.SLoRB_Weight = nn.Parameter(torch.zeros(Nout, rows, device=dev, dtype=self.weight.dtype),
                                             requires_grad=True)
        P = self.x_proj.data
        P.zero_()
        r = torch.arange(rows, device=dev)
        P[r[:, None], (r * k)[:, None] + torch.arange(k, device=dev)] = 1
        if self.SLoRB_init_type == "xavier":
            nn.init.xavier_uniform_(self.x_proj)
        else:
            pruned = (self.weight.detach() * (1.0 - self.mask.detach())).view(Nout, rows, k)
            if self.SLoRB_init_type == "mean":
                init = pruned.mean(dim=2)
            elif self.SLoRB_init_type == "sum":
                init = pruned.sum(dim=2)
            else:
                raise ValueError(f"Invalid SLoRB_init_type: {self.SLoRB_init_type}")
            self.SLoRB_Weight.data.copy_(init)

    # ---- hard projections ---------------------------------------------------
    def _effective_hard_type(self) -> str:
        hard_type = str(getattr(self, "hard_mask_type", "match") or "match")
        return self.mask_type if hard_type == "match" else hard_type

    def _hard_kind(self):
        """(SF_HARD_* kind, N, M) of this layer's hard projection."""
        t = self._effective_hard_type()
        if t == "none":
            return L.HARD_NONE, 2, 4
        if t == "unstructured":
            return L.HARD_THRESHOLD, 2, 4
        if t == "nm_2_4":
            return L.HARD_NM_TAIL_KEEP, 2, 4
        if t == "structured":
            return L.HARD_NM_STRICT, int(self.N), int(self.M)
        if t in _BLOCK_TYPES:  # not group-local: projected whole by _hard_mask_from_soft
            raise ValueError(f"hard_mask_type {t!r} has no per-group projection")
        raise ValueError(f"Invalid hard mask_type: {t}")

    def _is_block_hard(self) -> bool:
        return self._effective_hard_type() in _BLOCK_TYPES

    def _raw_hard_type(self) -> str:
        return str(getattr(self, "hard_mask_type", "match") or "match")

    def _block_sparsity_ratio(self, default: float) -> float:
        return float(getattr(self, "sparsity_ratio", default))

    @torch.no_grad()
    def _blockify_tensor(self, tensor: torch.Tensor) -> torch.Tensor:
        """(:460-507) every bs x bs block of the core takes its mean (block_sparse16/32 only)."""
        hard_type = self._raw_hard_type()
        if hard_type not in BM.BLOCK_SPARSE or tensor.dim() != 2:
            return tensor
        return BM.blockify_(tensor.detach().clone().contiguous(), hard_type)

    @torch.no_grad()
    def _flip_count(self, prev: torch.Tensor, now: torch.Tensor, counter: torch.Tensor) -> torch.Tensor:
        """Positions where the hard projections of prev and now differ (:1659-1661), added to counter."""
        if self._is_block_hard():
            hp, hn = self._hard_mask_from_soft(prev), self._hard_mask_from_soft(now)
            return K.hard_flip_count(hp, hn, L.HARD_THRESHOLD, counter=counter)
        kind, n, m = self._hard_kind()
        return K.hard_flip_count(prev, now, kind, n, m, counter=counter)

    @torch.no_grad()
    def _hard_mask_from_soft(self, soft_mask: torch.Tensor) -> torch.Tensor:
        """Project a soft mask to {0, 1} (:510-735) on the GPU."""
        t = self._effective_hard_type()
        if t == "none":
            return torch.ones_like(soft_mask)
        if t == "unstructured" or soft_mask.dim() == 1:
            return (soft_mask > 0.5).to(dtype=soft_mask.dtype)
        if t in _BLOCK_TYPES:  # block16 keeps round((1 - sr) 256) per tile; block_sparse keeps whole blocks
            return BM.hard_mask(soft_mask, t, self._block_sparsity_ratio(0.0 if t == "block16" else 0.5))
        kind, n, m = self._hard_kind()
        if kind == L.HARD_NM_STRICT and soft_mask.shape[1] % m != 0:
            raise ValueError(f"in_features ({soft_mask.shape[1]}) must be divisible by M ({m}).")
        return K.hard_mask(soft_mask.contiguous(), kind, n, m)

    # ---- forward --------------------------------------------------------------
    def _compute_weight_scale_factor(self) -> float:
        """(:799-827)"""
        t = self._effective_hard_type()
        if t == "none":
            return 1.0
        if t == "structured":
            N, M = int(self.N), int(self.M)
            if N <= 0 or M <= 0 or N >= M:
                return 1.0
            return float(M) / float(N)
        if t == "nm_2_4":
            return 2.0
        sr = float(self.sparsity_ratio)
        if sr <= 0.0 or sr >= 1.0:
            return 1.0
        return 1.0 / (1.0 - sr)

    def forward(self, x):
        """(:737-796): masked forward with STE backward, plus the SLoRB bypass."""
        if self.mode == "dense_forward" or self.mask_type == "none":
            mask_mode, hx, scale = "none", 1.0, 1.0
        elif self.mode == "sparse_forward":
            try:
                hx = float(getattr(self, "hardening_x", 1.0))
            except Exception:
                hx = 1.0
            finalized = bool(getattr(self, "_hardening_finalized", False))
            if hx >= 1.0 - 1e-6 or finalized:
                mask_mode = "soft"
            else:
                mask_mode = "mix"
            scale = 1.0
            if getattr(self.cfg, "weight_scaling", False) and hx < 1.0 - 1e-6:
                scale = 1.0 + (1.0 - hx) * (self._compute_weight_scale_factor() - 1.0)
        else:
            raise ValueError(f"Invalid mode: {self.mode}")
        slorb = self.SLoRB and hasattr(self, "x_proj")
        hard = None
        cache = self.__dict__.setdefault("_eff_cache", {})
        if mask_mode == "mix" and self._is_block_hard():
            kind, n, m = L.HARD_THRESHOLD, 2, 4
            # whole-tensor projection (:770), kept while the mask and the projection parameters are unchanged
            key = ("block", self.mask.data_ptr(), self.mask._version, self._effective_hard_type(),
                   self._block_sparsity_ratio(-1.0))
            if cache.get("hard_key") != key:
                cache.clear()
                cache["hard"], cache["hard_key"] = self._hard_mask_from_soft(self.mask), key
            hard = cache["hard"]
        elif mask_mode == "mix":
            kind, n, m = self._hard_kind()
            if kind == L.HARD_NM_STRICT and self.in_features % m != 0:
                raise ValueError(f"in_features ({self.in_features}) must be divisible by M ({m}).")
        else:
            kind, n, m = L.HARD_NONE, 2, 4
        return masked_linear(
            x, self.weight, self.bias, None if mask_mode == "none" else self.mask, mask_mode, hx, kind, n, scale,
            self.x_proj if slorb else None, self.SLoRB_Weight if slorb else None, 0.0, hard=hard, hard_m=m,
            cache=cache if hard is None else None,
        )

    # ---- WANDA calibration / grad EMA (off the paper path) -------------------
    @torch.no_grad()
    def add_batch(self, inp, out):
        """Input-norm accumulation for the wanda metric (:884-898)."""
        if self._is_placeholder("scaler_row"):
            return
        if len(inp.shape) == 2:
            inp = inp.unsqueeze(0)
        tmp = inp.shape[0]
        if len(inp.shape) == 3:
            inp = inp.reshape((-1, inp.shape[-1]))
        inp = inp.t()
        self.scaler_row.mul_(self.nsamples / (self.nsamples + tmp + 1e-8))
        self.nsamples += tmp
        inp = inp.float()
        self.scaler_row.add_((torch.norm(inp, p=2, dim=1) ** 2) / max(self.nsamples, 1))

    @torch.no_grad()
    def update_grad_hessian_ema(self, update_hessian_with_grad2: bool = True):
        """grad / grad^2 EMA for the movement metric (:901-923); returns early otherwise."""
        if self._is_placeholder("grad_ema") or self.weight.grad is None:
            return
        g = self.weight.grad.detach()
        if g.shape != self.grad_ema.shape:
            if g.numel() == self.grad_ema.numel():
                g = g.view_as(self.grad_ema)
            else:
                return
        b = float(self.cfg.beta)
        self.grad_ema.mul_(b).add_(g, alpha=1 - b)
        if update_hessian_with_grad2 and not self._is_placeholder("hessian_diag") and self.hessian_diag.shape == g.shape:
            self.hessian_diag.mul_(b).add_(g * g, alpha=1 - b)

    @torch.no_grad()
    def update_importance_ema(self):
        """Deprecated no-op kept for interface compatibility (:926-929)."""
        pass

    # ---- schedules (:932-985, :1603-1619): host scalars from sparseforge_amd.schedules ----
    def _hard_type_raw(self) -> str:
        return str(getattr(self, "hard_mask_type", "match") or "match")

    def _temperature(self, step: int) -> float:
        return SCH.temperature(self.cfg, self._hard_type_raw(), step)

    def _mask_update_period(self, step: int) -> int:
        return SCH.update_period(self.cfg, step)

    def _effective_sparsity(self, step: int) -> float:
        return SCH.effective_sparsity(self.cfg, self._hard_type_raw(), self.sparsity_ratio, step)

    def _beta_structural(self, step: int) -> float:
        return SCH.structural_mix(self.cfg, step)

    def _hardening_schedule(self, step: int) -> float:
        """hardening_x after an update at `step`."""
        return SCH.hardening_coefficient(self.cfg, step)

    # ---- device mask path --------------------------------------------------------
    def _mask_operands(self, scores_override: Optional[torch.Tensor] = None) -> K.MaskOperands:
        W = self.weight.detach()
        if scores_override is not None:
            return K.MaskOperands(weight=W, mask=self.mask.detach(), hessian=scores_override)
        H = None
        if not self._is_placeholder("hessian_diag") and self.hessian_diag.shape == W.shape:
            H = self.hessian_diag.data
        aux = None
        if self.mask_metric == "wanda" and not self._is_placeholder("scaler_row"):
            aux = self.scaler_row.data
        if self.mask_metric == "movement" and not self._is_placeholder("grad_ema") and self.grad_ema.shape == W.shape:
            aux = self.grad_ema.data
        # detach(), not .data: the kernels' in-place writes then bump the parameters' own version counters
        frozen = None if self._is_placeholder("frozen_mask_flags") else self.frozen_mask_flags.detach()
        return K.MaskOperands(weight=W, mask=self.mask.detach(), hessian=H, aux=aux, frozen=frozen)

    def _metric_code(self, ops: K.MaskOperands) -> int:
        metric = self.mask_metric
        code = L.METRIC.get(metric, L.METRIC["magnitude"])
        # missing operands fall back as in :1041-1079: W * W for hessian_obd, |W| for the others
        if metric in ("hessian_obd", "hessian_ratio", "hessian") and ops.hessian is None:
            return L.METRIC["magnitude"] if metric != "hessian_obd" else L.METRIC["weight_squared"]
        if metric in ("wanda", "movement") and ops.aux is None:
            return L.METRIC["magnitude"]
        return code

    def _score_dtype(self, ops: K.MaskOperands, metric_code: int) -> int:
        w = ops.weight.dtype
        if metric_code in (L.METRIC["hessian_obd"], L.METRIC["hessian_ratio"]):
            return _dtype_tag(torch.promote_types(w, ops.hessian.dtype))
        if metric_code == L.METRIC["hessian"]:
            return _dtype_tag(ops.hessian.dtype)
        if metric_code in (L.METRIC["wanda"], L.METRIC["movement"]):
            return _dtype_tag(torch.promote_types(w, ops.aux.dtype))
        return _dtype_tag(w)

    def _mask_params(self, step: int, ops: K.MaskOperands, metric_code: int, lambda_mid: float = 0.0,
                     with_update: bool = False) -> L.MaskParams:
        rows, cols = ops.weight.shape
        p = L.MaskParams()
        p.rows, p.cols = rows, cols
        p.metric = metric_code
        if self.mask_type == "unstructured":
            p.gate = L.GATE_UNSTRUCTURED
        elif self.mask_type == "structured":
            assert cols % int(self.M) == 0, f"in_features ({cols}) must be divisible by M ({int(self.M)})."
            p.gate = L.GATE_STRUCTURED_EXACT if getattr(self.cfg, "structured_exact", False) else L.GATE_STRUCTURED
        else:
            raise ValueError(f"Invalid mask_type: {self.mask_type}")
        p.n_keep, p.m_group = int(self.N), int(self.M)
        p.score_dtype = self._score_dtype(ops, metric_code)
        p.temperature = self._temperature(step)
        p.eps_metric = 1e-8
        p.movement_temp = max(float(self.cfg.temperature), 1e-8)
        p.beta_struct = self._beta_structural(step) if cols >= int(self.M) else 0.0
        if self._raw_hard_type() in BM.BLOCK_SPARSE:  # no N:M mix for block_sparse (:1203-1205)
            p.beta_struct = 0.0
        p.has_frozen = int(ops.frozen is not None)
        if with_update:
            # block hard types count flips from whole-tensor projections (_flip_count)
            kind, hn, hm = (L.HARD_THRESHOLD, 2, 4) if self._is_block_hard() else self._hard_kind()
            p.hard_kind, p.hard_n, p.hard_m = kind, hn, hm
            lam = float(lambda_mid or 0.0)
            p.penalty = L.PENALTY_NONE
            p.penalty_coef = 0.0
            if lam != 0.0:
                mode = str(getattr(self.cfg, "mask_penalty_mode", "mid") or "mid")
                if mode in BM.BLOCK_SIZE:  # the staged update builds the target (or falls back to mid)
                    mode = "target"
                if mode == "nm_2_4" and (cols // 4) * 4 == 0:
                    mode = "mid"
                if mode == "structured_topn" and cols % int(self.M) != 0:
                    mode = "mid"
                p.penalty = {"nm_2_4": L.PENALTY_NM_2_4, "structured_topn": L.PENALTY_STRUCTURED_TOPN,
                             "mid": L.PENALTY_MID, "target": L.PENALTY_TARGET}.get(mode, L.PENALTY_NONE)
                p.penalty_coef = float(self.mask_penalty_lr) * lam
            try:
                d = float(self.cfg.mask_binarize_decay) if getattr(self.cfg, "mask_binarize_decay", None) is not None else 0.0
            except Exception:
                d = 0.0
            p.binarize = d
            p.mask_lr = float(self.cfg.mask_lr)
            low, high = float(self.cfg.freeze_low), float(self.cfg.freeze_high)
            p.apply_freeze = int(low > 0.0 or high < 1.0)
            p.freeze_low, p.freeze_high = low, high
            p.snap_high = int(step >= 2000)
        return p

    def _sample_size(self, n: int) -> Optional[int]:
        """Size of the tau sample over n scores, or None when the reference takes every score (:991-996)."""
        m = int(self.cfg.tau_sample_size) if self.cfg.tau_sample_size is not None else n
        return m if (m > 0 and n > m) else None

    def _sample_seed(self, n: int) -> Optional[int]:
        """Seed of this update's tau sample (drawn from torch's default CPU generator), or None."""
        if self._sample_size(n) is None:
            return None
        return int(torch.randint(0, 1 << 62, (1,)).item())

    def _sample_indices(self, n: int, device) -> Optional[torch.Tensor]:
        """The tau sample.  The reference draws torch.randint(0, n, (m,)) (:993) and takes a quantile of
        the sampled scores, which does not depend on the sample's order: the library draws the same law
        in non-decreasing order (sf_sample_indices_sorted), which lets the batched update read the
        sampled scores from its statistics pass instead of gathering them."""
        seed = self._sample_seed(n)
        if seed is None:
            return None
        return draw_samples(self._sample_size(n), [n], [seed], device)[0]

    def _gate_inputs(self, step: int, ops: K.MaskOperands, metric_code: int, p: L.MaskParams,
                     sample_idx: Optional[torch.Tensor] = None):
        """Score statistics and (unstructured) tau on the device."""
        stats = K.score_stats(p, ops)
        tau = None
        if p.gate == L.GATE_UNSTRUCTURED:
            if sample_idx is None:
                sample_idx = self._sample_indices(ops.weight.numel(), ops.weight.device)
            tau = K.tau_quantile(p, ops, stats, self._effective_sparsity(step), sample_idx)
        return stats, tau

    @torch.no_grad()
    def _tau_unstructured(self, scores: torch.Tensor, sparsity: float) -> torch.Tensor:
        """torch.quantile over a random sample of `scores` (:987-1015), on the device."""
        s = scores.detach().contiguous()
        s2 = s.view(1, -1) if s.dim() != 2 else s
        ops = K.MaskOperands(weight=s2, mask=s2, hessian=s2)
        p = L.MaskParams()
        p.rows, p.cols = s2.shape
        p.metric = L.METRIC["hessian"]
        p.score_dtype = _dtype_tag(s.dtype)
        stats = torch.tensor([0.0, 1.0], dtype=torch.float32, device=s.device)
        idx = self._sample_indices(s.numel(), s.device)
        tau = K.tau_quantile(p, ops, stats, float(sparsity), idx)[0]
        if getattr(self, "_in_summon_context", False):
            return tau
        try:
            import torch.distributed as dist

            if dist.is_available() and dist.is_initialized():
                t = tau.clone()
                dist.all_reduce(t, op=dist.ReduceOp.SUM)
                t.div_(dist.get_world_size())
                tau = t
        except Exception:
            pass
        return tau

    @torch.no_grad()
    def compute_gate_target(self, step: int, sample_idx: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Soft-mask target G in [0, 1] (:1018-1239).  `sample_idx` optionally injects the tau sample."""
        if (not self.change_mask) or (self.mask_type == "none"):
            return torch.ones_like(self.mask)
        if self.weight.numel() == 0:
            return self.mask
        ops = self._mask_operands()
        code = self._metric_code(ops)
        p = self._mask_params(step, ops, code)
        stats, tau = self._gate_inputs(step, ops, code, p, sample_idx)
        return self._gate(step, ops, p, stats, tau)

    def _gate(self, step: int, ops: K.MaskOperands, p: L.MaskParams, stats, tau) -> torch.Tensor:
        """G on the device: elementwise, or the block_sparse block gate, then the block_sparse blockify."""
        g_dtype = torch.bfloat16 if p.score_dtype == L.DT_BF16 else torch.float32
        hard_type = self._raw_hard_type()
        if hard_type not in BM.BLOCK_SPARSE:
            return K.gate_target(p, ops, stats, tau, g_dtype)
        ob, ib = BM.core_blocks(ops.weight.shape, BM.BLOCK_SIZE[hard_type])
        if self.mask_type == "unstructured" and ob > 0 and ib > 0:  # (:1122-1154)
            pz = L.MaskParams.from_buffer_copy(p)
            pz.gate, pz.beta_struct, pz.has_frozen = L.GATE_ZSCORE, 0.0, 0
            z = K.gate_target(pz, ops, stats, None, g_dtype)
            G = BM.block_gate(z, hard_type, self._effective_sparsity(step), p.temperature, ops.mask, ops.frozen)
        else:
            G = K.gate_target(p, ops, stats, tau, g_dtype)
        return BM.blockify_(G, hard_type)  # (:1237)

    @torch.no_grad()
    def update_mask(self, step: int, lambda_mid: float = 0.0, sample_idx: Optional[torch.Tensor] = None):
        """Periodic mask EMA update (:1242-1666) as one fused device pass."""
        prep = self._prepare_update(step, lambda_mid)
        if prep is None:
            return
        ops, p, code = prep
        stats, tau = self._gate_inputs(step, ops, code, p, sample_idx)
        flips = torch.zeros(1, dtype=torch.int64, device=self.mask.device)
        if self._staged_update(p):
            self._update_mask_staged(step, ops, p, stats, tau, flips)
        else:
            K.update_mask(p, ops, stats, tau, flips)
        self._finish_update(step, flips)

    def _staged_update(self, p: L.MaskParams) -> bool:
        """Block hard types and block penalty modes take the multi-pass update."""
        return self._is_block_hard() or self._raw_hard_type() in BM.BLOCK_SPARSE or p.penalty == L.PENALTY_TARGET

    def _finish_update(self, step: int, flips: torch.Tensor) -> None:
        """Host state after an update: hardening schedule (:1644-1656) and the flip counters (:1659-1664)."""
        self.hardening_x = self._hardening_schedule(step)
        # the flip count stays on the device until someone reads it (int() syncs)
        self.weight.flipped_mask = flips[0]
        self.weight.init_flipped_mask = 0
        self.weight.mask = self.mask

    def _prepare_update(self, step: int, lambda_mid: float = 0.0):
        """The gating of update_mask (:1242-1287): None when this step leaves the mask alone, else
        (operands, device parameters, metric code) of the update."""
        if self.mask.numel() == 0:
            return None
        if self.mask.dim() != 2:
            if not getattr(self, "_warned_mask_dim_at_entry", False):
                warnings.warn(f"[update_mask] mask.dim()={self.mask.dim()}, shape={self.mask.shape}. "
                              f"Expected 2D. weight.shape={self.weight.shape}. Skipping this layer.")
                self._warned_mask_dim_at_entry = True
            return None
        if self.weight.shape != self.mask.shape:
            if not getattr(self, "_warned_fsdp_shape_mismatch", False):
                warnings.warn(f"[update_mask] Shape mismatch: weight.shape={self.weight.shape}, "
                              f"mask.shape={self.mask.shape}. Skipping this layer's mask update.")
                self._warned_fsdp_shape_mismatch = True
            return None
        if (not self.change_mask) or (self.mask_type == "none"):
            self.weight.flipped_mask = 0
            self.weight.init_flipped_mask = 0
            return None
        if step < int(self.cfg.sparsity_warmup_steps):
            return None
        K_ = max(1, int(self._mask_update_period(step)))
        if step % K_ != 0:
            return None
        ops = self._mask_operands()
        code = self._metric_code(ops)
        p = self._mask_params(step, ops, code, lambda_mid, with_update=True)
        return ops, p, code


    def _update_mask_staged(self, step: int, ops: K.MaskOperands, p: L.MaskParams, stats, tau, flips) -> None:
        """update_mask for the block hard types and block penalty modes, in passes:
        G (elementwise or per block, :1018-1239) -> penalty target (:1298-1529) -> penalty, clamp,
        binarisation, EMA (sf_apply_gate) -> blockify (:1598-1601) -> freeze (:1621-1642) -> flips."""
        mask = self.mask.detach()
        prev = mask.clone()
        G = self._gate(step, ops, p, stats, tau)
        target = None
        if p.penalty == L.PENALTY_TARGET:
            mode = str(getattr(self.cfg, "mask_penalty_mode", "mid") or "mid")
            sr = self._block_sparsity_ratio(0.0 if mode == "block16" else 0.5)
            target = BM.penalty_target(mode, G, mask, sr)
            if target is None:  # no full block: the reference falls back to 'mid'
                p.penalty = L.PENALTY_MID
        block_sparse = self._raw_hard_type() in BM.BLOCK_SPARSE
        K.apply_gate(p, G, target, mask, ops.frozen, do_freeze=not block_sparse)
        if block_sparse:
            BM.blockify_(mask, self._raw_hard_type())
            K.freeze_mask(p, mask, ops.frozen)
        self._flip_count(prev, mask, flips)


class Distill_Model(torch.nn.Module):
    """Student/teacher distillation wrapper (legacy/sparse_modeling.py:1669-1838).

    Beyond the reference: with top > 0 the KL is that from the teacher's `top` largest logits and the probability of all
    other tokens together (distill.top_kl_loss); forward also takes such a record of the teacher's (distill.TopLogits) as
    teacher_top, and then runs no teacher, which may be None.  Without a teacher and a record the KL is 0, and with top > 0
    the call is refused."""

    def __init__(self, model, teacher=None, output_hidden_state=False, top=0):
        super().__init__()
        self.student = model
        self.teacher = teacher
        self.top = int(top)
        self.student.config.output_hidden_state = output_hidden_state
        self.output_hidden_state = output_hidden_state
        if teacher is not None:
            self.teacher.config.output_hidden_state = output_hidden_state
            self.teacher.eval()

    def _teacher_forward(self, idx, targets):
        with torch.no_grad():
            try:
                tdev = next(self.teacher.parameters()).device
            except Exception:
                tdev = idx.device
            idx_t = idx.to(device=tdev) if idx.device != tdev else idx
            targets_t = None
            if targets is not None:
                targets_t = targets.to(device=tdev) if targets.device != tdev else targets
            return self.teacher(idx_t, targets_t)

    def forward(self, idx, targets=None, teacher_top=None):
        if teacher_top is not None:
            from .distill import top_kl_loss

            if self.output_hidden_state:
                raise ValueError("Distill_Model: a record of the teacher's logits has no hidden states")
            student_logits, task_loss, _ = self.student(idx, targets)
            return student_logits, task_loss, None, top_kl_loss(student_logits, teacher_top)
        if self.teacher is None:
            if self.top:
                raise ValueError(f"Distill_Model: the KL from the teacher's top {self.top} needs a teacher or a record")
            student_logits, task_loss, _ = self.student(idx, targets)
            return student_logits, task_loss, None, torch.tensor(0.0, device=idx.device)
        if self.output_hidden_state:
            student_logits, task_loss, student_hidden = self.student(idx, targets)
            teacher_logits, _, teacher_hidden = self._teacher_forward(idx, targets)
            if teacher_logits.device != student_logits.device:
                teacher_logits = teacher_logits.to(device=student_logits.device, dtype=student_logits.dtype)
            if teacher_hidden is not None and student_hidden is not None and len(teacher_hidden) == len(student_hidden):
                teacher_hidden = [t.to(device=student_logits.device, dtype=student_logits.dtype) for t in teacher_hidden]
            if student_hidden is not None and teacher_hidden is not None:
                layerwise = self.layerwise_loss(student_hidden, teacher_hidden)
            else:
                layerwise = 0.0
            return student_logits, task_loss, layerwise, self._kl(student_logits, teacher_logits)
        student_logits, task_loss, _ = self.student(idx, targets)
        teacher_logits, _, _ = self._teacher_forward(idx, targets)
        if teacher_logits.device != student_logits.device:
            teacher_logits = teacher_logits.to(device=student_logits.device, dtype=student_logits.dtype)
        return student_logits, task_loss, None, self._kl(student_logits, teacher_logits)

    def _kl(self, student_logits, teacher_logits):
        if not self.top:
            return self.kl_loss(student_logits, teacher_logits)
        from .distill import top_kl_loss, top_logits

        return top_kl_loss(student_logits, top_logits(teacher_logits, self.top))

    def kl_loss(self, student_logits, teacher_logits, temperature=2):
        """KL(P_teacher || Q_student) at temperature T, logits clamped to +-100 (:1749-1828)."""
        from .distill import chunked_kl_loss

        return chunked_kl_loss(student_logits, teacher_logits, temperature)

    def layerwise_loss(self, student_hidden_states, teacher_hidden_states):
        """(:1830-1838)"""
        loss = 0.0
        eps = torch.finfo(torch.bfloat16).eps
        for s, t in zip(student_hidden_states, teacher_hidden_states):
            loss += (s - t).pow(2).mean() / (t.pow(2).mean() + eps)
        return loss
