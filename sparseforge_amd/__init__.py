"""sparseforge_amd: MI355X-native sparse-training hot path of SparseForge.

Drop-in modules mirroring liuhanzuo/SparseForge legacy/:
  sparse_modeling  SparseLinearConfig, SparseLinear, FusedMaskedLinearSTE, Distill_Model
  utils            mask-op functions (calculate_model_mask, update_hessian_hutchinson, ...)
  adamw            AdamW with the mask-aware decay
  block_sparse     convert_to_block_sparse, BlockSparseLinear (block-sparse-16 GEMM)
Beside them, what generating with a finalized model needs:
  rotary           rotary_embed, rotary_cos_sin, RotaryScaling (rotary positions)
  kv_cache         KVCache8 (keys and values in 8 bits, attention over them)
  logits           process_logits (penalties, bias, grammar masks)
  generate         Generator, generate (the three together on a LlamaDecoder)
All tensor work runs in the HIP library libsparseforge_amd.so (gfx950).
"""
from . import _lib  # noqa: F401

__all__ = ["_lib"]
