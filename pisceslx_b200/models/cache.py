"""Paged KV cache.

The reference keeps Python lists of per-layer block objects and concatenates them on every read
(model/core/cache.py:535-868, read path :824-835); its unified manager is lossy by default (H2O,
quantisation, eviction; cache.py:1886-2038).  Here the cache is two device tensors per layer
``[num_blocks, block_size, n_kv_head, head_dim]`` plus an int32 block table per sequence; the decode kernel
reads pages in place.  ``YvPagedLayeredCache`` keeps the same pages, tables and free list for layer runs that each store
what they need (keys and values of sizes of their own, or one latent row per token), and gives pages back once every
layer's window has passed them.  The cache is exact; eviction policies (LRU of whole sequences, sliding window) are
opt-in helpers that only edit block tables.  Two more options are opt-in and lossy.  With ``dtype`` float8_e4m3fn ``YvPagedKVCache`` holds
keys and values as 8-bit codes and one exponent byte for each token and head (``ops.cache``), a little over half the bytes of
bf16.  With ``attention_window`` a token attends to the last ``attention_window`` tokens and to the ``first_tokens`` first of its
sequence (streaming attention: the first tokens carry much of every softmax), and pages that only hold others are given back.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Tuple

import numpy as np
import torch


RELEASED = -1      # table entry of a page that was given back because no later token can see it


@dataclass
class YvCacheConfig:
    block_size: int = 64
    num_blocks: int = 1024
    max_blocks_per_seq: int = 2048
    dtype: torch.dtype = torch.bfloat16
    sliding_window: Optional[int] = None      # keep only the last N tokens addressable (opt-in, lossy)
    attention_window: Optional[int] = None    # tokens attend to the last N tokens, their own included (opt-in, lossy) ...
    first_tokens: int = 0                     # ... and to the first ones of their sequence


class YvBlockAllocator:
    """Free-list allocator of cache pages with reference counts (prefix sharing)."""

    def __init__(self, num_blocks: int):
        self.num_blocks = num_blocks
        self.free: List[int] = list(range(num_blocks - 1, -1, -1))
        self.refs: Dict[int, int] = {}

    def available(self) -> int:
        return len(self.free)

    def alloc(self) -> int:
        if not self.free:
            raise MemoryError("paged KV cache is out of blocks")
        b = self.free.pop()
        self.refs[b] = 1
        return b

    def share(self, b: int) -> int:
        self.refs[b] += 1
        return b

    def release(self, b: int) -> None:
        self.refs[b] -= 1
        if self.refs[b] == 0:
            del self.refs[b]
            self.free.append(b)


class YvPagedKVCache:
    """Block pool for all layers of one model replica plus per-sequence block tables (host side)."""

    def __init__(self, n_layer: int, n_kv_head: int, head_dim: int, cfg: YvCacheConfig, device: torch.device):
        self.cfg, self.device = cfg, device
        self.n_layer, self.hk, self.d = n_layer, n_kv_head, head_dim
        shape = (cfg.num_blocks, cfg.block_size, n_kv_head, head_dim)
        if cfg.attention_window is not None and (cfg.attention_window < 1 or cfg.first_tokens < 0):
            raise ValueError(f"a window of {cfg.attention_window} tokens and {cfg.first_tokens} first ones")
        if cfg.attention_window is None and cfg.first_tokens:
            raise ValueError("first_tokens are those that stay visible beside an attention_window")
        if cfg.attention_window is not None and cfg.sliding_window is not None:
            raise ValueError("attention_window masks keys where they lie, sliding_window moves them: one of the two")
        self.fp8 = cfg.dtype == torch.float8_e4m3fn
        if self.fp8 and cfg.sliding_window is not None:
            raise ValueError("8-bit pages are read through whole tables, which sliding_window cuts: attention_window masks keys instead")
        if self.pages_only and not self.continues:
            raise ValueError(f"8-bit pages, and windows, are for heads of 64 or 128 numbers and pages of a multiple of 16 tokens, bf16 or 8 "
                             f"bits: heads of {head_dim}, pages of {cfg.block_size}, {cfg.dtype}")
        page = lambda: torch.zeros(shape, dtype=torch.uint8, device=device).view(cfg.dtype) if self.fp8 else \
            torch.zeros(shape, dtype=cfg.dtype, device=device)
        self.k = [page() for _ in range(n_layer)]
        self.v = [page() for _ in range(n_layer)]
        scale = lambda: torch.zeros(cfg.num_blocks, n_kv_head, cfg.block_size, dtype=torch.uint8, device=device)
        self.k_scale = [scale() for _ in range(n_layer)] if self.fp8 else []
        self.v_scale = [scale() for _ in range(n_layer)] if self.fp8 else []
        self.alloc = YvBlockAllocator(cfg.num_blocks)
        self.tables: Dict[int, List[int]] = {}       # seq id -> physical blocks
        self.lengths: Dict[int, int] = {}
        self.layer_offset = 0                         # first global layer index held by this pipeline stage
        # tokens (the query's own included) that the widest layer still reads; None = every token stays addressable
        self.reach: Optional[int] = cfg.attention_window

    @property
    def pages_only(self) -> bool:
        """Whether attention has to go through ``ops.cache`` (8-bit pages, or a window over them)."""
        return self.fp8 or self.cfg.attention_window is not None

    @property
    def continues(self) -> bool:
        """Whether ``ops.cache`` reads these pages on their device, so that a prompt's later portion can attend to earlier ones.  Tables
        that ``sliding_window`` cuts do not say where they begin."""
        return self.cfg.sliding_window is None and (torch.device(self.device).type != "cuda" or (
            self.d in (64, 128) and self.cfg.block_size % 16 == 0 and self.cfg.dtype in (torch.bfloat16, torch.float8_e4m3fn)))

    def scales(self, idx: int) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """Exponent bytes of a layer's keys and values in 8 bits, else (None, None)."""
        at = idx - self.layer_offset
        return (self.k_scale[at], self.v_scale[at]) if self.fp8 else (None, None)

    def read(self, seq_id: int, idx: int, lo: int = 0, hi: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys (as rotated at their positions) and values of a sequence's tokens lo .. hi - 1 in one layer [hi - lo, hk * d]: a
        prefix to hand to another cache, or to look at."""
        slots = self.slots(seq_id, lo, self.lengths[seq_id] if hi is None else hi)
        at = torch.from_numpy(slots).to(self.device)
        k, v = self.layer(idx)
        if self.fp8:
            from ..ops import cache as C
            return C.kv_cache_read_fp8(k, v, *self.scales(idx), at.int())
        return k.view(-1, self.hk * self.d)[at], v.view(-1, self.hk * self.d)[at]

    def layer(self, idx: int) -> Tuple[torch.Tensor, torch.Tensor]:
        return self.k[idx - self.layer_offset], self.v[idx - self.layer_offset]

    def bytes(self) -> int:
        return 2 * self.n_layer * self.k[0].numel() * self.k[0].element_size() + sum(t.numel() for t in self.k_scale + self.v_scale)

    # ---- sequence management (host) ---------------------------------------------------------------
    def add_sequence(self, seq_id: int) -> None:
        self.tables[seq_id] = []
        self.lengths[seq_id] = 0

    def free_sequence(self, seq_id: int) -> None:
        for b in self.tables.pop(seq_id, []):
            if b != RELEASED:
                self.alloc.release(b)
        self.lengths.pop(seq_id, None)

    def release_passed(self, seq_id: int) -> int:
        """Give back the pages that no token from here on can see (all layers windowed; see ``reach``).  Their table
        entries stay as placeholders, so that page i keeps holding tokens ``i * block_size ...``.  One page of slack
        is kept for callers that step back a few tokens.  Returns the number of pages freed."""
        if self.reach is None:
            return 0
        bs, tbl = self.cfg.block_size, self.tables[seq_id]
        last = (self.lengths[seq_id] - self.reach + 1 - bs) // bs          # pages below this one are out of reach
        kept = -(-self.cfg.first_tokens // bs)                             # pages of the first tokens
        freed = 0
        for i in range(min(last, len(tbl)) - 1, kept - 1, -1):
            if tbl[i] == RELEASED:
                break                                                     # everything in front of it has gone before
            self.alloc.release(tbl[i])
            tbl[i] = RELEASED
            freed += 1
        return freed

    def fork(self, src: int, dst: int) -> None:
        """Share all full blocks of ``src`` with ``dst`` (prefix caching / beam search)."""
        self.tables[dst] = [b if b == RELEASED else self.alloc.share(b) for b in self.tables[src]]
        self.lengths[dst] = self.lengths[src]

    def can_append(self, seq_id: int, n_tokens: int) -> bool:
        need = self._blocks_needed(seq_id, n_tokens)
        return need <= self.alloc.available()

    def _blocks_needed(self, seq_id: int, n_tokens: int) -> int:
        bs = self.cfg.block_size
        have = len(self.tables[seq_id])
        total = (self.lengths[seq_id] + n_tokens + bs - 1) // bs
        return max(0, total - have)

    def append_slots(self, seq_id: int, n_tokens: int) -> List[int]:
        """Reserve room for ``n_tokens`` new tokens; returns their flat slot ids (block * block_size + offset)."""
        bs = self.cfg.block_size
        self.release_passed(seq_id)
        for _ in range(self._blocks_needed(seq_id, n_tokens)):
            self.tables[seq_id].append(self.alloc.alloc())
        start = self.lengths[seq_id]
        tbl = self.tables[seq_id]
        slots = [tbl[(start + i) // bs] * bs + (start + i) % bs for i in range(n_tokens)]
        self.lengths[seq_id] = start + n_tokens
        return slots

    def slots(self, seq_id: int, lo: int, hi: int) -> np.ndarray:
        """Flat slot ids of the tokens lo .. hi - 1 (which must not have been given back)."""
        bs = self.cfg.block_size
        pos = np.arange(lo, hi)
        pages = np.asarray(self.tables[seq_id], dtype=np.int64)[pos // bs]
        if pages.size and int(pages.min()) < 0:
            raise IndexError(f"sequence {seq_id}: tokens {lo}..{hi - 1} reach into released pages")
        return pages * bs + pos % bs

    def block_table_tensor(self, seq_ids: List[int], width: Optional[int] = None) -> torch.Tensor:
        width = width or max(1, max(len(self.tables[s]) for s in seq_ids))
        t = torch.zeros(len(seq_ids), width, dtype=torch.int32)
        for i, s in enumerate(seq_ids):
            tbl = self.tables[s]
            if self.cfg.sliding_window is not None:
                keep = (self.cfg.sliding_window + self.cfg.block_size - 1) // self.cfg.block_size + 1
                tbl = tbl[-keep:]
            t[i, : len(tbl)] = torch.tensor(tbl, dtype=torch.int32)
        return t.to(self.device, non_blocking=True)

    def seq_lens_tensor(self, seq_ids: List[int]) -> torch.Tensor:
        return torch.tensor([self.lengths[s] for s in seq_ids], dtype=torch.int32).to(self.device, non_blocking=True)

    # ---- checkpoint / restore (reference cache.py:2394-2430) ------------------------------------------------
    def state(self) -> Dict[str, object]:
        return {"tables": {k: list(v) for k, v in self.tables.items()}, "lengths": dict(self.lengths),
                "k": [t.cpu() for t in self.k], "v": [None if t is None else t.cpu() for t in self.v],
                "k_scale": [t.cpu() for t in self.k_scale], "v_scale": [t.cpu() for t in self.v_scale]}

    def load_state(self, st: Dict[str, object]) -> None:
        pairs = []
        for mine, saved in ((self.k, st["k"]), (self.v, st["v"]), (self.k_scale, st.get("k_scale", [])),
                            (self.v_scale, st.get("v_scale", []))):
            if len(mine) != len(saved):                                        # type: ignore[arg-type]
                raise ValueError("the saved cache holds its keys and values in another form")
            for t, src in zip(mine, saved):                                    # type: ignore[arg-type]
                if t is not None:
                    if src is None or t.shape != src.shape:
                        raise ValueError(f"saved pages of {None if src is None else tuple(src.shape)} for {tuple(t.shape)}")
                    if t.dtype != src.dtype and torch.float8_e4m3fn in (t.dtype, src.dtype):
                        raise ValueError(f"a saved cache of {src.dtype} for one of {t.dtype}")
                    pairs.append((t, src))
        # nothing has been touched so far
        self.tables = {int(k): list(v) for k, v in st["tables"].items()}      # type: ignore[union-attr]
        self.lengths = {int(k): int(v) for k, v in st["lengths"].items()}     # type: ignore[union-attr]
        used = {b for t in self.tables.values() for b in t if b != RELEASED}
        self.alloc = YvBlockAllocator(self.cfg.num_blocks)
        self.alloc.free = [b for b in range(self.cfg.num_blocks - 1, -1, -1) if b not in used]
        self.alloc.refs = {b: sum(b in t for t in self.tables.values()) for b in used}
        for t, src in pairs:
            t.copy_(src)


class YvPagedLayeredCache(YvPagedKVCache):
    """Pages whose contents differ from layer run to layer run.  Layout i is ``{"row": n}`` (one row of n numbers per
    token) or ``{"heads": g, "dim": d, "vdim": e}`` (keys ``[num_blocks, block_size, g, d]`` and values ``[.., g, e]``)."""

    def __init__(self, layouts: List[Dict[str, int]], cfg: YvCacheConfig, device: torch.device, reach: Optional[int] = None):
        if cfg.dtype == torch.float8_e4m3fn or cfg.attention_window is not None:
            raise ValueError("layered models bring windows of their own and read bf16 or fp32 pages")
        self.fp8, self.k_scale, self.v_scale = False, [], []
        self.cfg, self.device = cfg, device
        self.n_layer = len(layouts)
        self.hk = max(m.get("heads", 1) for m in layouts)
        self.d = max(m["row"] if "row" in m else max(m["dim"], m["vdim"]) for m in layouts)
        page = lambda *tail: torch.zeros(cfg.num_blocks, cfg.block_size, *tail, dtype=cfg.dtype, device=device)
        self.k = [page(m["row"]) if "row" in m else page(m["heads"], m["dim"]) for m in layouts]
        self.v = [None if "row" in m else page(m["heads"], m["vdim"]) for m in layouts]
        self.alloc = YvBlockAllocator(cfg.num_blocks)
        self.tables, self.lengths = {}, {}
        self.layer_offset = 0
        self.reach = reach

    @property
    def continues(self) -> bool:
        return True                                   # these layers read pages in ways of their own

    def rows(self, idx: int) -> torch.Tensor:
        if self.v[idx - self.layer_offset] is not None:
            raise TypeError("this layer stores keys and values: use layer()")
        return self.k[idx - self.layer_offset]

    def layer(self, idx: int):
        if self.v[idx - self.layer_offset] is None:
            raise TypeError("this layer stores one row per token: use rows()")
        return super().layer(idx)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.k + self.v if t is not None)


def cache_for_model(cfg, device: torch.device, num_blocks: int, block_size: Optional[int] = None, tp_size: int = 1,
                    n_layer: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, attention_window: Optional[int] = None,
                    first_tokens: int = 0) -> YvPagedKVCache:
    """``dtype`` float8_e4m3fn, ``attention_window`` and ``first_tokens``: see ``YvCacheConfig``."""
    if tp_size > 1 and attention_window is not None:
        # there prompts are padded at their end, and a prompt's last row is taken for its last token
        raise ValueError("attention_window: not with tensor parallelism")
    cc = YvCacheConfig(block_size=block_size or cfg.kv_cache_block_size, num_blocks=num_blocks, dtype=dtype,
                       attention_window=attention_window, first_tokens=first_tokens)
    if cfg.layer_specs:
        from .registry import cache_layout
        layouts, reach = cache_layout(cfg)
        return YvPagedLayeredCache(layouts, cc, device, reach)
    return YvPagedKVCache(n_layer or cfg.n_layer, cfg.n_kv_head // tp_size, cfg.head_dim, cc, device)
