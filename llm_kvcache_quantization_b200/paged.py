"""Paged KV cache: one pool of fixed-size pages per layer, a page table per sequence, sequences of any length in a batch.

Where the contiguous caches of `cache.py` hold one length for all rows and reallocate as they grow, a `PagedKVCache` takes
its memory once and hands out pages: sequences join (`add_sequence`) and leave (`free_sequence`) between steps, each with
its own length.  Per layer and step it makes the same two calls: the fused quantize-append of the new tokens
(`ops.paged_append`, same codes and scales as the contiguous caches, bit for bit) and the fused decode attention
(`ops.span_attn`), with no host synchronisation.  An object also serves as the engine behind the patched attention forward
(`engine.INT8CacheWrapperContainer`): `append` / `fused_decode` / `get_kv` / `get_seq_len` have the contiguous caches'
meaning, for the rows in `sequences`.

No counterpart in the reference (its caches are contiguous, src/cache/protocol.py:30-63).
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import ops
from .cache import _new_stats

KV_FORMATS = ("fp16", "int8", "int4", "int4_asym")


class PagedKVCache:
    """`num_pages` pages of `page_size` tokens per layer, shared by all sequences of the cache.

    kv_format: "fp16", "int8", "int4" (symmetric groups, `clip_percentile` of each group's magnitudes or the static tables
    [L, Hkv, G] when given) or "int4_asym" (min / max groups with zero-points).  `window` / `sinks` make `fused_decode` attend
    only the last `window` and the first `sinks` tokens of each sequence.  page_size must be a multiple of 16.
    """

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, *, page_size: int = 64,
                 kv_format: str = "int8", group_size: int = 128, clip_percentile: float = 99.9,
                 max_pages_per_seq: Optional[int] = None, window: Optional[int] = None, sinks: int = 0,
                 static_k_scale: Optional[Tensor] = None, static_v_scale: Optional[Tensor] = None,
                 inv_tau: Optional[Tensor] = None, use_attn_temperature: bool = True, device="cuda",
                 dtype: torch.dtype = torch.float16):
        for name, val in (("num_layers", num_layers), ("num_pages", num_pages), ("num_kv_heads", num_kv_heads)):
            if val <= 0:
                raise ValueError(f"{name} must be > 0, got {val}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size must be a multiple of 16, got {page_size}")
        if kv_format not in KV_FORMATS:
            raise ValueError(f"kv_format must be one of {KV_FORMATS}, got {kv_format!r}")
        group_size = head_dim if group_size == -1 or kv_format == "fp16" else group_size
        if group_size <= 0 or head_dim % group_size or group_size % 8:
            raise ValueError(f"head_dim {head_dim} must be divisible by group_size {group_size}, a multiple of 8")
        if window is not None and (window < 1 or sinks < 0):
            raise ValueError(f"window must be >= 1 and sinks >= 0, got {window}, {sinks}")
        if window is None and sinks:
            raise ValueError("sinks go with a window")
        if (static_k_scale is None) != (static_v_scale is None):
            raise ValueError("static_k_scale and static_v_scale must be given together")
        if static_k_scale is not None and kv_format not in ("int8", "int4"):
            raise ValueError("static scales are for the symmetric formats int8 and int4")
        if not 0.0 < clip_percentile <= 100.0:
            raise ValueError(f"clip_percentile must be in (0, 100], got {clip_percentile}")
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self.num_kv_heads, self.head_dim, self.kv_format, self.group_size = num_kv_heads, head_dim, kv_format, group_size
        self.clip_percentile, self.window, self.sinks = clip_percentile, window, sinks
        self.device, self.dtype = torch.device(device), dtype
        self.inv_tau, self.use_attn_temperature = inv_tau, use_attn_temperature
        self.decode_attn_impl = "triton_fused"             # the name the patched forward dispatches on
        self.max_pages_per_seq = min(num_pages, max_pages_per_seq or num_pages)
        self._static = None
        if static_k_scale is not None:
            G = head_dim // group_size
            for name, t in (("static_k_scale", static_k_scale), ("static_v_scale", static_v_scale)):
                if tuple(t.shape) != (num_layers, num_kv_heads, G):
                    raise ValueError(f"{name} must be [L={num_layers}, Hkv={num_kv_heads}, G={G}], got {tuple(t.shape)}")
            self._static = tuple(t.to(device=self.device, dtype=t.dtype if t.dtype in (torch.float16, torch.float32)
                                      else torch.float32).contiguous() for t in (static_k_scale, static_v_scale))
        width = head_dim // 2 if kv_format.startswith("int4") else head_dim
        pdt = torch.float16 if kv_format == "fp16" else torch.int8
        self._pools: List[Dict[str, Tensor]] = []
        for _ in range(num_layers):
            # zero-filled: rows of a page that nothing was written to yet are never attended, but they are copied into
            # on-chip memory with their neighbours
            pool = {n: torch.zeros(num_pages, num_kv_heads, page_size, width, dtype=pdt, device=self.device) for n in "kv"}
            names = ((), ("ks", "vs"), ("ks", "vs"), ("ks", "vs", "kz", "vz"))[KV_FORMATS.index(kv_format)]
            for n in names:
                pool[n] = torch.zeros(num_pages, num_kv_heads, page_size, head_dim // group_size, dtype=torch.float16,
                                      device=self.device)
            self._pools.append(pool)
        self._free = list(range(num_pages - 1, -1, -1))    # page 0 is handed out first
        self._pages: Dict[int, List[int]] = {}             # sequence -> its pages
        self._lens: Dict[int, int] = {}
        self._order: List[int] = []                        # the rows of a batch
        self._next_id = 0
        self._step: Optional[Tuple[Tensor, Tensor, Tensor, int, Optional[Tensor]]] = None
        self._step_layer = 0                               # layers appended so far in the current step
        self._step_tokens = 0
        self.decode_stats = _new_stats()

    # ---- sequences
    @property
    def sequences(self) -> Tuple[int, ...]:
        """The sequences that form the batch rows, in row order."""
        return tuple(self._order)

    @property
    def num_free_pages(self) -> int:
        return len(self._free)

    def add_sequence(self) -> int:
        """A new, empty sequence, the last row of the batch from the next step on."""
        self._between_steps("add_sequence")
        sid, self._next_id = self._next_id, self._next_id + 1
        self._pages[sid], self._lens[sid] = [], 0
        self._order.append(sid)
        self._step = None
        return sid

    def free_sequence(self, seq: int) -> None:
        """Drop a sequence and return its pages.  Work that was enqueued on the stream the cache is used on may still read
        them: pages are reused in the same stream order."""
        self._between_steps("free_sequence")
        if seq not in self._pages:
            raise ValueError(f"unknown sequence {seq}")
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lens[seq]
        self._order.remove(seq)
        self._step = None

    def get_seq_lens(self) -> Tuple[int, ...]:
        return tuple(self._lens[s] for s in self._order)

    def get_seq_len(self) -> int:
        return max(self.get_seq_lens(), default=0)

    def _between_steps(self, what: str) -> None:
        if 0 < self._step_layer < self.num_layers:
            raise ValueError(f"{what} in the middle of a step: layer {self._step_layer} of {self.num_layers} has not been "
                             "appended yet")

    # ---- one step
    def _not_captured(self) -> None:
        # pages and lengths are the host's, and the tables of a step live until the next one
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise ValueError("a step of a paged cache cannot be captured into a CUDA graph: use paged_append and "
                             "decode_attn_paged with tables of your own")

    def _begin(self, batch: int, tokens: int, new_lens: Optional[Sequence[int]]) -> None:
        """Reserve the pages of the step's tokens and upload its tables.  Nothing changes if the pool is too small."""
        self._between_steps("a new step")
        if batch != len(self._order):
            raise ValueError(f"the batch has {batch} rows, the cache {len(self._order)} sequences")
        counts = [tokens] * batch if new_lens is None else [int(x) for x in new_lens]
        if len(counts) != batch or any(c < 0 or c > tokens for c in counts):
            raise ValueError(f"new_lens must be {batch} counts in [0, {tokens}], got {counts}")
        want = []
        for s, c in zip(self._order, counts):
            pages = -(-(self._lens[s] + c) // self.page_size)
            if pages > self.max_pages_per_seq:
                raise ValueError(f"sequence {s} would need {pages} pages, max_pages_per_seq is {self.max_pages_per_seq}")
            want.append(pages - len(self._pages[s]))
        if sum(want) > len(self._free):
            raise ValueError(f"page pool exhausted: {sum(want)} pages needed, {len(self._free)} free of {self.num_pages}")
        start = [self._lens[s] for s in self._order]
        for s, c, w in zip(self._order, counts, want):
            for _ in range(w):
                self._pages[s].append(self._free.pop())
            self._lens[s] += c
        cols = max((len(self._pages[s]) for s in self._order), default=0) or 1
        # start, count and length of every row, then its table: one upload per step
        rows = [[st, c, self._lens[s]] + self._pages[s] + [-1] * (cols - len(self._pages[s]))
                for s, st, c in zip(self._order, start, counts)]
        host = torch.tensor(rows, dtype=torch.int32).reshape(batch, 3 + cols)
        if self.device.type == "cuda":
            host = host.pin_memory()
        meta = host.to(self.device, non_blocking=True)
        cols3 = meta[:, :3].t().contiguous()
        even = all(c == tokens for c in counts)
        self._step = (meta[:, 3:], cols3[0], cols3[2], self.get_seq_len(), None if even else cols3[1])
        self._step_layer = 0

    def _check_layer(self, layer_id: int) -> Dict[str, Tensor]:
        if layer_id < 0 or layer_id >= self.num_layers:
            raise ValueError(f"layer_id {layer_id} out of range [0, {self.num_layers})")
        return self._pools[layer_id]

    def append(self, layer_id: int, k: Tensor, v: Tensor, new_lens: Optional[Sequence[int]] = None) -> None:
        """Quantize and append new tokens [B, Hkv, T, D], row i to sequence `sequences[i]`.  The call for layer 0 opens the
        step: with `new_lens` (host counts, 0..T) row i takes only its first new_lens[i] tokens (prompts padded on the
        right; 0: the row sits out); the other layers follow in order with the same counts."""
        pool = self._check_layer(layer_id)
        if k.ndim != 4 or k.shape != v.shape:
            raise ValueError(f"k/v must be 4D [B,H,T,D] of one shape, got {tuple(k.shape)} / {tuple(v.shape)}")
        if k.shape[1] != self.num_kv_heads or k.shape[3] != self.head_dim:
            raise ValueError(f"expected [B, {self.num_kv_heads}, T, {self.head_dim}], got {tuple(k.shape)}")
        if not k.is_cuda or not v.is_cuda:
            raise ValueError("this cache quantizes with a CUDA kernel; CPU tensors are not supported")
        self._not_captured()
        if layer_id == 0:
            self._begin(k.shape[0], k.shape[2], new_lens)
            self._step_tokens = k.shape[2]
        elif layer_id != self._step_layer:
            raise ValueError(f"layers are appended in order: expected layer {self._step_layer}, got {layer_id}")
        elif k.shape[0] != len(self._order) or k.shape[2] != self._step_tokens:
            raise ValueError(f"expected {len(self._order)} rows of {self._step_tokens} tokens as in layer 0, got {tuple(k.shape)}")
        table, start, _, _, counts = self._step
        st = (None, None) if self._static is None else (self._static[0][layer_id], self._static[1][layer_id])
        if k.shape[0] and k.shape[2]:
            ops.paged_append(k, v, pool["k"], pool["v"], pool.get("ks"), pool.get("vs"), table, start, counts,
                             k_zp=pool.get("kz"), v_zp=pool.get("vz"), k_static=st[0], v_static=st[1],
                             clip_percentile=float(self.clip_percentile))
        self._step_layer = layer_id + 1

    def _live_step(self, layer_id: int):
        pool = self._check_layer(layer_id)
        self._not_captured()
        if self._step is None or layer_id >= self._step_layer:
            raise ValueError(f"nothing was appended to layer {layer_id} in this step")
        return pool, self._step

    def fused_decode(self, layer_id: int, q: Tensor, sm_scale: Optional[float] = None, inv_tau: Optional[Tensor] = None,
                     out: Optional[Tensor] = None) -> Tensor:
        """Attention of q [B, Hq, D] over everything cached for the layer, row i over sequence `sequences[i]` (inside the
        window, if the cache has one); an empty sequence gives zeros."""
        pool, (table, _, lens, longest, _) = self._live_step(layer_id)
        original = q.dtype
        res = ops.span_attn(q.to(torch.float16), pool["k"], pool["v"], pool.get("ks"), pool.get("vs"), lens, sm_scale,
                            k_zp=pool.get("kz"), v_zp=pool.get("vz"), block_table=table, window=self.window,
                            sinks=self.sinks, max_ctx=longest, inv_tau=inv_tau, out=out)
        return res if original == torch.float16 else res.to(original)

    def get_kv(self, layer_id: int) -> Tuple[Tensor, Tensor]:
        """(k, v) [B, Hkv, longest, D] of all rows as the cache holds them, zeros behind each row's length."""
        pool, (table, _, lens, longest, _) = self._live_step(layer_id)
        k, v = ops.paged_read(pool["k"], pool["v"], pool.get("ks"), pool.get("vs"), table, None, longest, lens,
                              head_dim=self.head_dim, k_zp=pool.get("kz"), v_zp=pool.get("vz"))
        return k.to(self.dtype), v.to(self.dtype)

    def clear(self) -> None:
        """Drop all sequences, keep the pools."""
        self._step_layer = 0
        for s in list(self._order):
            self.free_sequence(s)

    def get_memory_mb(self) -> float:
        return sum(t.numel() * t.element_size() for p in self._pools for t in p.values()) / (1024 * 1024)

    # ---- decode statistics (read by the patched forward's callers)
    def record_fused_decode(self, layer_id: int, decode_impl: str) -> None:
        st = self.decode_stats
        st["fused_decode_calls"] = int(st["fused_decode_calls"]) + 1
        hits = st["layer_hits"]
        hits[str(layer_id)] = int(hits.get(str(layer_id), 0)) + 1

    def get_decode_stats(self) -> Dict[str, object]:
        return {k: (dict(v) if isinstance(v, dict) else int(v)) for k, v in self.decode_stats.items()}

    def __repr__(self) -> str:
        return (f"{type(self).__name__}(num_layers={self.num_layers}, kv_format={self.kv_format!r}, "
                f"sequences={len(self._order)}, free_pages={len(self._free)}/{self.num_pages}, "
                f"memory={self.get_memory_mb():.2f}MB)")
