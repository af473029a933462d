"""Generating text with a LlamaDecoder, before or after its projections are finalized or packed 2:4.

A step takes the new tokens of every sequence through the model once: queries and keys are turned to their positions
(rotary.rotary_embed), keys and values go into a cache of 8-bit codes and the queries attend over it
(kv_cache.KVCache8), and the last token's logits are penalised, biased and masked (logits.process_logits) before the
next one is picked or drawn (logits.sample_logits).  The reference has no such path: it scores text by running whole sequences
(legacy/eval_wiki_ppl.py:548-651).
"""
from __future__ import annotations

import torch

from .kv_cache import KVCache8
from .llama import LlamaDecoder, swiglu
from .logits import process_logits, sample_logits
from .rotary import rotary_cos_sin, rotary_embed


class Generator:
    """A LlamaDecoder (bfloat16, on the GPU) with the caches of a batch of sequences of at most `capacity` tokens.

    A step calls the norms and projections of the model's layers itself, with the cached attention between them: forward
    hooks of these run, those of a layer or of the model do not."""

    def __init__(self, model: LlamaDecoder, batch: int, capacity: int):
        weight = model.embed_tokens.weight
        if not weight.is_cuda:
            raise RuntimeError(f"sparseforge_amd runs on the GPU only; the model is on {weight.device}")
        if weight.dtype != torch.bfloat16:
            raise TypeError(f"Generator: the model is {weight.dtype} (bfloat16 only)")
        c = model.config
        self.model, self.batch, self.device = model, batch, weight.device
        self.cache = KVCache8(batch, c.num_attention_heads, c.head_dim, capacity, len(model.layers), weight.device)
        self.cos, self.sin = rotary_cos_sin(self.cache.capacity, c.head_dim, c.rope_theta, c.rope_scaling, weight.device)

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, counts: torch.Tensor | None = None) -> torch.Tensor:
        """tokens [B, n], the first counts[b] (int32 [B], n where None) of a row real, any ids in the others -> the logits
        [B, V] after each row's last real token (of a row without one: without meaning)."""
        m, cache = self.model, self.cache
        if tokens.dim() != 2 or tokens.shape[0] != self.batch or tokens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"Generator.step: tokens must be ids [{self.batch}, n], got {tokens.dtype} "
                             f"{tuple(tokens.shape)}")
        if tokens.device != self.device:
            raise ValueError(f"Generator.step: tokens are on {tokens.device}, the model on {self.device}")
        B, n = tokens.shape
        cache.extend(n, counts)
        positions = cache.starts[:, None]
        if n > 1:
            # rows past a sequence's tokens, whose results are not used, stay inside the tables
            positions = (positions + torch.arange(n, device=self.device, dtype=torch.int32)).clamp_(
                max=cache.capacity - 1)
        if counts is not None:  # ids that pad a row may be none of the embedding's (-1, say)
            real = torch.arange(n, device=self.device) < counts[:, None]
            tokens = torch.where(real, tokens, tokens.clamp(0, m.config.vocab_size - 1))
        h = m.embed_tokens(tokens)
        for i, layer in enumerate(m.layers):
            a, f = layer.self_attn, layer.mlp
            x = layer.input_layernorm(h)
            q, k, v = (p(x).view(B, n, layer.heads, -1) for p in (a.q_proj, a.k_proj, a.v_proj))
            q, k = rotary_embed(q, k, self.cos, self.sin, positions)
            cache.append(k, v, i)
            h = h + a.o_proj(cache.attend(q, layer=i))
            x = layer.post_attention_layernorm(h)
            h = h + f.down_proj(swiglu(f.gate_proj(x), f.up_proj(x)))
        if n == 1:
            h = h[:, 0]
        elif counts is None:
            h = h[:, -1]
        else:
            h = h[torch.arange(B, device=self.device), (counts.long() - 1).clamp_(0, n - 1)]
        return m.lm_head(m.norm(h))


@torch.no_grad()
def generate(model: LlamaDecoder, prompts: torch.Tensor, new_tokens: int, lengths: torch.Tensor | None = None, *,
             repetition=1.0, presence=0.0, frequency=0.0, bias: torch.Tensor | None = None, allowed=None, pick=None,
             end_token: int | None = None, chunk: int = 2048, temperature=None, top_k=0, top_p=1.0, min_p=0.0,
             generator: torch.Generator | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Continue prompts [B, S] (the first lengths[b], at least one, of a row; what pads a row is not looked at) by up to
    new_tokens tokens each.

    Returns (tokens int64 [B, S + new_tokens], lengths int32 [B]): each prompt with its continuation, and how many
    tokens that is; what lies past a row's length has no meaning.  The penalties, bias and allowed are process_logits',
    with the prompt and the answer so far as the history;
    allowed may be a function of (tokens, lengths) that gives the mask of a step.  pick turns logits [B, V] into ids
    [B]: the most likely token (the lowest id among equals) where None.  With a temperature tokens are drawn instead, by
    logits.sample_logits with top_k, top_p and min_p and random numbers from `generator` (the device's own where None),
    one for each sequence and token.  A sequence stops after end_token, and where its mask or bias lets nothing follow,
    a drawn one also where its logits hold a NaN; the logits that pick sees of one that has stopped are zeros.  Prompts
    are taken `chunk` tokens at a time."""
    if prompts.dim() != 2 or prompts.shape[1] < 1 or prompts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"generate: prompts must be ids [B, S], got {prompts.dtype} {tuple(prompts.shape)}")
    if pick is not None and temperature is not None:
        raise ValueError("generate: pick and a temperature both say how tokens are chosen")
    if temperature is None:
        given = {"top_k": (top_k, 0), "top_p": (top_p, 1.0), "min_p": (min_p, 0.0)}
        unused = [n for n, (x, none) in given.items() if torch.is_tensor(x) or x != none]
        unused += ["generator"] if generator is not None else []
        if unused:
            raise ValueError(f"generate: {', '.join(unused)} without a temperature, which draws tokens")
    if new_tokens < 0 or chunk < 1:
        raise ValueError(f"generate: {new_tokens} new tokens, chunks of {chunk}")
    B, S = prompts.shape
    gen = Generator(model, B, S + max(new_tokens, 1))
    dev = gen.device
    if lengths is None:
        lengths = torch.full((B,), S, dtype=torch.int32, device=dev)
    elif lengths.shape != (B,) or lengths.dtype != torch.int32 or lengths.device != dev:
        raise ValueError(f"generate: lengths must be int32 [{B}] on {dev}")
    elif bool(((lengths < 1) | (lengths > S)).any()):
        raise ValueError(f"generate: lengths must lie in 1 .. {S}, got {lengths.tolist()}")
    lengths = lengths.clone()
    tokens = torch.zeros(B, S + new_tokens, dtype=torch.int64, device=dev)
    tokens[:, :S] = prompts
    logits = None
    for at in range(0, S, chunk):
        n = min(chunk, S - at)
        counts = (lengths - at).clamp_(0, n)
        out = gen.step(tokens[:, at:at + n], counts)
        logits = out if logits is None else torch.where((counts > 0)[:, None], out, logits)
    alive = torch.ones(B, dtype=torch.int32, device=dev)
    shaped = allowed is not None or bias is not None
    drawn = temperature is not None
    stops = shaped or drawn or end_token is not None
    for i in range(new_tokens):
        mask = allowed(tokens, lengths) if callable(allowed) else allowed
        logits = process_logits(logits, tokens, lengths, repetition=repetition, presence=presence,
                                frequency=frequency, bias=bias, allowed=mask, out=logits)
        if shaped:
            alive = alive * ~(logits == float("-inf")).all(-1)
        if drawn:
            uniform = torch.rand(B, device=dev, generator=generator)
            ids = sample_logits(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
            alive = alive * (ids >= 0)
        elif pick is None:
            ids = logits.argmax(-1)
        else:
            ids = pick(logits.masked_fill(alive[:, None] == 0, 0.0) if stops else logits)
        at = lengths.long()[:, None]
        tokens.scatter_(1, at, torch.where(alive[:, None] > 0, ids[:, None].long(), tokens.gather(1, at)))
        lengths += alive
        if end_token is not None:
            alive = alive * (ids != end_token)
        if i + 1 < new_tokens:
            logits = gen.step(ids[:, None], alive if stops else None)
    return tokens, lengths
