"""A cache of keys and values held in 8 bits, and attention over it (sf_kv8_*).

For generating with a model: the reference evaluates and samples by running the whole sequence again
(legacy/eval_wiki_ppl.py:548-651), so there is no counterpart in it.

64 consecutive tokens of one sequence and head are a block, held as int8 codes with one scale for its keys and one for
its values; a sequence's last block stays in bf16 until it is whole (the header's sf_kv8_cache has the format).  A step
of a model with `layers` layers is

    cache.extend(n, counts)            # once: room for n more tokens of every sequence (counts[b] of them real)
    cache.append(k, v, layer)          # each layer: their keys and values
    out = cache.attend(q, layer=layer) # each layer: their queries over everything so far, themselves included

k, v are [B, n, Hk, D], q is [B, n, H, D] in bfloat16, H a multiple of Hk (query head h reads key-value head
h / (H / Hk)), D a multiple of 8 up to 256.  Forward only.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L
from . import profiling as _prof
from .kernels import _written

BLOCK = 64  # tokens that share a scale


class KVCache8:
    """Keys and values of `batch` sequences of at most `capacity` tokens (rounded up to whole blocks) for `layers`
    layers.  `ends` [batch] int32 holds the sequences' lengths on the device, `bound` what the host knows them to be
    at most (exact when every counts[b] is n).

    A step may be captured in a graph and replayed: the lengths advance on the device, and the kernels read them and
    stay inside the capacity.  `bound`, which sizes attend's launch, is that of the capture: set it to the length that
    the replays will reach before capturing."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, capacity: int, layers: int = 1, device="cuda"):
        if min(batch, kv_heads, capacity, layers) < 1:
            raise ValueError("KVCache8: batch, kv_heads, capacity and layers must be positive")
        if head_dim < 8 or head_dim > 256 or head_dim % 8:
            raise ValueError(f"KVCache8: head_dim {head_dim} must be a multiple of 8 up to 256")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError(f"sparseforge_amd runs on the GPU only; got device {device} (no CPU path exists)")
        blocks = -(-capacity // BLOCK)
        self.batch, self.kv_heads, self.head_dim, self.layers = batch, kv_heads, head_dim, layers
        self.capacity = blocks * BLOCK
        rows = -(-head_dim // 64) * 64 * BLOCK
        shape = (layers, batch, kv_heads, blocks)

        def empty(*shape, dtype):
            return torch.empty(shape, dtype=dtype, device=self.device)

        self.k_codes, self.v_codes = empty(*shape, rows, dtype=torch.int8), empty(*shape, rows, dtype=torch.int8)
        self.k_scales, self.v_scales = empty(*shape, dtype=torch.float32), empty(*shape, dtype=torch.float32)
        self.k_tail = empty(layers, batch, kv_heads, rows, dtype=torch.bfloat16)
        self.v_tail = empty(layers, batch, kv_heads, rows, dtype=torch.bfloat16)
        self.starts = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.ends = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.bound = 0
        self._new = 0  # tokens of the step under way
        self._descs = [self._desc(i, blocks) for i in range(layers)]
        self._refs = [ctypes.byref(d) for d in self._descs]

    def _desc(self, i: int, blocks: int) -> L.Kv8Cache:
        d = L.Kv8Cache()
        for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail"):
            setattr(d, name, getattr(self, name)[i].data_ptr())
        d.starts, d.ends = self.starts.data_ptr(), self.ends.data_ptr()
        d.batch, d.kv_heads, d.head_dim, d.blocks = self.batch, self.kv_heads, self.head_dim, blocks
        return d

    def reset(self) -> None:
        """Every sequence empty again."""
        self.starts.zero_()
        self.ends.zero_()
        self.bound = self._new = 0

    def extend(self, n: int, counts: torch.Tensor | None = None) -> None:
        """Begin a step of n tokens a sequence: of counts[b] (int32 [batch] on the device, 0 .. n), the first of its
        rows, where given.  The capacity is checked against `bound`."""
        if n < 1:
            raise ValueError(f"KVCache8.extend: {n} tokens")
        if self.bound + n > self.capacity:
            raise ValueError(f"KVCache8.extend: {n} tokens after up to {self.bound}, the capacity is {self.capacity}")
        if counts is not None:
            if L.require_device(counts) != self.ends.device:
                raise ValueError("KVCache8.extend: counts are on another device")
            if counts.dtype != torch.int32 or counts.shape != (self.batch,):
                raise ValueError(f"KVCache8.extend: counts must be int32 [{self.batch}]")
        dev = self.ends.device
        with _prof.region("sf_kv8_extend", 12 * self.batch, "B", dev):
            L.check(L.lib().sf_kv8_extend(self._refs[0], n, L.ptr(counts), L.stream(dev)), "sf_kv8_extend")
        _written(self.starts, self.ends)  # a backward may have saved starts as positions
        self.bound += n
        self._new = n

    def _rows(self, t: torch.Tensor, name: str, heads: int | None) -> torch.Tensor:
        """t as the kernels read it: contiguous heads, rows at 16-byte aligned addresses."""
        if t.get_device() != self.ends.get_device():
            L.require_device_only(t)
            raise ValueError(f"KVCache8: {name} is on {t.device}, the cache on {self.ends.device}")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"KVCache8: {name} is {t.dtype} (bfloat16 only)")
        shape = t.shape
        if len(shape) != 4 or shape[0] != self.batch or shape[3] != self.head_dim or \
                (shape[2] != heads if heads else shape[2] % self.kv_heads or shape[2] == 0):
            raise ValueError(f"KVCache8: {name} {tuple(shape)} does not go with {self.batch} sequences, "
                             f"{self.kv_heads} heads of {self.head_dim}")
        if shape[1] != self._new:
            raise ValueError(f"KVCache8: {name} holds {shape[1]} tokens a sequence, the step has {self._new}")
        sb, ss, sh, sd = t.stride()
        if sd != 1 or (sb | ss | sh) % 8 or t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def append(self, k: torch.Tensor, v: torch.Tensor, layer: int = 0) -> None:
        """The step's keys and values [B, n, Hk, D] of one layer, once in a step: where they complete a block, its kept
        rows give way to those after it, and a second call would code these instead."""
        k, v = self._rows(k, "k", self.kv_heads), self._rows(v, "v", self.kv_heads)
        dev = self.ends.device
        with _prof.region("sf_kv8_append", 3 * k.numel() * k.element_size(), "B", dev):
            L.check(L.lib().sf_kv8_append(self._refs[layer], k.data_ptr(), *k.stride()[:3], v.data_ptr(),
                                          *v.stride()[:3], self._new, L.stream(dev)), "sf_kv8_append")

    def attend(self, q: torch.Tensor, scale: float | None = None, window: int = 0, layer: int = 0) -> torch.Tensor:
        """Attention of the step's queries q [B, n, H, D] over the keys up to their own (the last `window` of them if
        window > 0), after append -> [B, n, H * D].  scale: D^-0.5 where none is given.  Rows past counts[b] are 0."""
        q = self._rows(q, "q", None)
        B, n, H, D = q.shape
        if scale is None:
            scale = D ** -0.5
        dev = self.ends.device
        lib = L.lib()
        out = torch.empty((B, n, H * D), dtype=q.dtype, device=dev)
        size = lib.sf_kv8_attend_workspace_size(B, self.kv_heads, H, D, n, self.bound)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        with _prof.region("sf_kv8_attend", 4 * self.bound * n * B * H * D, "FLOP", dev):
            L.check(lib.sf_kv8_attend(self._refs[layer], q.data_ptr(), *q.stride()[:3], n, H, scale, window, self.bound,
                                      out.data_ptr(), L.ptr(ws), size, L.stream(dev)), "sf_kv8_attend")
        return out

    def values(self, first: int | torch.Tensor = 0, tokens: int | None = None, layer: int = 0):
        """The keys and values that the cache stands for, float32 [B, tokens, Hk, D] each, from position `first` (a
        number, or int32 [batch] on the device) on; 0 past a sequence's end.  tokens: up to `bound` where none given."""
        if tokens is None:
            tokens = max(0, self.bound - first) if isinstance(first, int) else self.bound
        if not 0 <= tokens <= self.capacity:
            raise ValueError(f"KVCache8.values: {tokens} tokens, the capacity is {self.capacity}")
        dev = self.ends.device
        at = None
        if not isinstance(first, int):
            if L.require_device(first) != dev or first.dtype != torch.int32 or first.shape != (self.batch,):
                raise ValueError(f"KVCache8.values: first must be a number or int32 [{self.batch}] on {dev}")
            at, first = first, 0
        shape = (self.batch, tokens, self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=torch.float32, device=dev)
        v = torch.empty(shape, dtype=torch.float32, device=dev)
        with _prof.region("sf_kv8_values", 10 * k.numel(), "B", dev):
            L.check(L.lib().sf_kv8_values(self._refs[layer], L.ptr(at), first, tokens, k.data_ptr(),
                                          v.data_ptr(), L.stream(dev)), "sf_kv8_values")
        return k, v
