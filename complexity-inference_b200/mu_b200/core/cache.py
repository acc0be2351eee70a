"""Paged KV cache: a GPU block pool with MuPagedCache-compatible bookkeeping.

Pool layout (one allocation): ``[num_layers][2][num_blocks][num_kv_heads]
[block_size][head_dim]``, so the K (or V) tile of one (block, kv head) is a
contiguous ``block_size * head_dim`` run for the attention kernels, and a
layer's K and V are plain 4-D views.  With dtype float8_e4m3fn the pool holds
e4m3 codes and ``scales`` ``[num_layers][2][num_blocks][num_kv_heads]`` f32 the
scale of each (block, head): a cached value is code * scale, at half the bytes.

Block bookkeeping reproduces mu_inference/core/cache.py:257-462 exactly:
the free list starts as ``list(range(N))`` and is popped from the end
(LIFO); ``allocate`` takes one block even for an empty request; a new block
is taken only when a token arrives while the last block is full; ``free``
returns blocks in table order.  Block tables and slot mappings therefore
match the reference allocator bit for bit.

One deliberate difference: the reference advances a request's position on
every ``append`` call, i.e. once per layer (cache.py:340, 374), so a
multi-layer model spreads one token over several slots.  Here slots are
reserved once per token per step (:meth:`PagedKVCache.reserve`) and shared
by all layers; the reference-style ``append(request_id, layer_idx, k, v)``
keeps its signature and reuses the slots reserved by the layer-0 call.

``fork`` gives a request a second continuation: full blocks are shared (counted
in ``block_refs``; nobody writes a full block), the last, partly filled one is
copied on the device with its scales.  ``compact`` moves the live blocks to the
front of the pool.  Neither has a counterpart in the reference.
"""

from __future__ import annotations

import threading
from collections import Counter
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .config import MuConfig
from .mu import mu_clamp


class PagedKVCache:
    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, block_size: int = 16,
                 max_num_blocks: int = 2048, dtype: torch.dtype = torch.bfloat16,
                 device: str = "cuda", mu_config: Optional[MuConfig] = None):
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.block_size = block_size
        self.max_num_blocks = max_num_blocks
        self.dtype = dtype
        self.device = device
        self.mu_config = mu_config or MuConfig()
        self.quantized = dtype == torch.float8_e4m3fn
        self.block_pool = torch.zeros(num_layers, 2, max_num_blocks, num_kv_heads, block_size,
                                      head_dim, dtype=dtype, device=device)
        self.scales: Optional[torch.Tensor] = None
        if self.quantized:
            self.scales = torch.ones(num_layers, 2, max_num_blocks, num_kv_heads, device=device)
        self.free_blocks: List[int] = list(range(max_num_blocks))
        self.request_blocks: Dict[str, List[int]] = {}
        self.request_pos: Dict[str, int] = {}
        self.block_refs: Dict[int, int] = {}  # holders of blocks that several requests share
        self._pending: Dict[str, np.ndarray] = {}
        self._lock = threading.RLock()

    # ---- device views ------------------------------------------------------
    def k_cache(self, layer: int) -> torch.Tensor:
        return self.block_pool[layer, 0]

    def v_cache(self, layer: int) -> torch.Tensor:
        return self.block_pool[layer, 1]

    def k_scale(self, layer: int) -> Optional[torch.Tensor]:
        return None if self.scales is None else self.scales[layer, 0]

    def v_scale(self, layer: int) -> Optional[torch.Tensor]:
        return None if self.scales is None else self.scales[layer, 1]

    # ---- reference API (cache.py:311-453) -----------------------------------
    def allocate(self, request_id: str) -> bool:
        """Give a new request its first block (LIFO pop); False when full."""
        with self._lock:
            if not self.free_blocks:
                return False
            self.request_blocks[request_id] = [self.free_blocks.pop()]
            self.request_pos[request_id] = 0
            return True

    def reserve(self, request_id: str, num_tokens: int) -> Optional[np.ndarray]:
        """Slots (block*block_size + offset) for the next ``num_tokens`` tokens.

        All-or-nothing: returns None (state unchanged) when the request is
        unknown or the pool cannot hold the tokens."""
        with self._lock:
            blocks = self.request_blocks.get(request_id)
            if blocks is None:
                return None
            bs = self.block_size
            pos = self.request_pos[request_id]
            n = int(num_tokens)
            if n <= 0:
                return np.empty(0, dtype=np.int32)
            first = min(n, bs - pos) if pos < bs else 0
            rest = n - first
            need = (rest + bs - 1) // bs
            if need > len(self.free_blocks):
                return None
            out = np.empty(n, dtype=np.int32)
            if first:
                out[:first] = blocks[-1] * bs + pos + np.arange(first, dtype=np.int32)
            if need:
                new = [self.free_blocks.pop() for _ in range(need)]
                blocks.extend(new)
                idx = np.arange(rest, dtype=np.int32)
                out[first:] = np.asarray(new, dtype=np.int32)[idx // bs] * bs + idx % bs
                self.request_pos[request_id] = rest - (need - 1) * bs
            else:
                self.request_pos[request_id] = pos + first
            return out

    def blocks_needed(self, request_id: str, num_tokens: int) -> int:
        """New blocks a reserve(request_id, num_tokens) would take."""
        pos = self.request_pos.get(request_id, 0)
        first = min(num_tokens, self.block_size - pos) if pos < self.block_size else 0
        return (num_tokens - first + self.block_size - 1) // self.block_size

    def append(self, request_id: str, layer_idx: int, keys: torch.Tensor,
               values: torch.Tensor) -> int:
        """Reference-compatible append of [1, T, Hkv, D] keys/values for one layer.

        Layer 0 reserves T new slots; other layers write the same slots.
        mu_clamp is applied when enabled with apply_to_kv_cache, as in
        cache.py:342-355.  This API path is a convenience for callers of the
        reference interface; the forward step writes the cache with the
        fused RoPE+append kernel instead.  Returns the sequence length, or
        -1 on failure."""
        with self._lock:
            if request_id not in self.request_blocks:
                return -1
            T = keys.shape[1]
            slots = self._pending.get(request_id)
            if layer_idx == 0 or slots is None or len(slots) != T:
                slots = self.reserve(request_id, T)
                if slots is None:
                    return -1
                self._pending[request_id] = slots
            if self.mu_config.enabled and self.mu_config.apply_to_kv_cache:
                c = self.mu_config
                keys = mu_clamp(keys, c.mu, c.clamp_min, c.clamp_max)
                values = mu_clamp(values, c.mu, c.clamp_min, c.clamp_max)
            if self.quantized:
                for i, x in enumerate((keys, values)):
                    self._store_quantized(layer_idx, i, x[0].float(), slots)
                return self.get_seq_len(request_id)
            s = torch.as_tensor(slots, dtype=torch.long, device=self.block_pool.device)
            blk, off = s // self.block_size, s % self.block_size
            self.block_pool[layer_idx, 0, blk, :, off] = keys[0].to(self.dtype)
            self.block_pool[layer_idx, 1, blk, :, off] = values[0].to(self.dtype)
            return self.get_seq_len(request_id)

    def _store_quantized(self, layer: int, kv: int, x: torch.Tensor, slots: np.ndarray) -> None:
        """x [T, Hkv, D] f32 into the codes and scales of a layer's K or V, block by block:
        the arithmetic of the fused append (muk_rope_kv_append_fp8)."""
        codes, scale = self.block_pool[layer, kv], self.scales[layer, kv]
        bs = self.block_size
        at = 0
        while at < len(slots):
            blk, end = int(slots[at]) // bs, at
            while end < len(slots) and int(slots[end]) // bs == blk:
                end += 1
            rows = x[at:end].to(codes.device)                       # [n, Hkv, D]
            off = torch.as_tensor(np.asarray(slots[at:end]) % bs, dtype=torch.long,
                                  device=codes.device)
            amax = rows.abs().amax((0, 2))
            m, e = torch.frexp(amax)                                # 448 = 0.875 * 2^9
            e = torch.where(amax > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -60))
            new = torch.exp2(e.clamp(-60, 60).float())
            bad = ~torch.isfinite(amax)
            if int(slots[at]) % bs != 0:                            # the block keeps its older rows
                old = scale[blk]
                bad |= old.isnan()
                new = torch.maximum(new, old)
                ratio = torch.where(bad, torch.ones_like(old), old / new)
                codes[blk] = (codes[blk].float() * ratio[:, None, None]).to(codes.dtype)
            y = torch.where(bad[None, :, None], torch.zeros_like(rows), rows / new[None, :, None])
            codes[blk][:, off] = y.clamp(-448, 448).to(codes.dtype).transpose(0, 1)
            scale[blk] = torch.where(bad, torch.full_like(new, float("nan")), new)
            at = end

    def get(self, request_id: str, layer_idx: int
            ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """All cached K, V of a request/layer as [1, T, Hkv, D] (cache.py:377-413)."""
        with self._lock:
            blocks = self.request_blocks.get(request_id)
            if not blocks:
                return None, None
            n = self.get_seq_len(request_id)
            if n == 0:
                return None, None
            idx = torch.as_tensor(blocks, dtype=torch.long, device=self.block_pool.device)
            kv = []
            for i in range(2):
                x = self.block_pool[layer_idx, i, idx]
                if self.quantized:  # the values that the codes stand for
                    x = x.float() * self.scales[layer_idx, i, idx][:, :, None, None]
                x = x.transpose(1, 2).reshape(-1, self.num_kv_heads, self.head_dim)[:n]
                kv.append(x.unsqueeze(0))
            return kv[0], kv[1]

    def get_seq_len(self, request_id: str) -> int:
        with self._lock:
            blocks = self.request_blocks.get(request_id)
            if not blocks:
                return 0
            return (len(blocks) - 1) * self.block_size + self.request_pos[request_id]

    def block_table(self, request_id: str) -> List[int]:
        return self.request_blocks.get(request_id, [])

    def held_blocks(self, *request_ids: str) -> int:
        """Blocks that freeing all of these requests would give back (those that no
        other request shares)."""
        with self._lock:
            tables = [self.request_blocks.get(r, []) for r in request_ids]
            if not self.block_refs:
                return sum(len(t) for t in tables)
            n = Counter(b for t in tables for b in t)
            return sum(1 for b, k in n.items() if k == self.block_refs.get(b, 1))

    def free(self, request_id: str) -> None:
        with self._lock:
            blocks = self.request_blocks.pop(request_id, [])
            if self.block_refs:
                blocks = [b for b in blocks if self._drop_ref(b)]
            self.free_blocks.extend(blocks)
            self.request_pos.pop(request_id, None)
            self._pending.pop(request_id, None)

    def _drop_ref(self, block: int) -> bool:
        """One holder less; True when that was the last one."""
        n = self.block_refs.get(block)
        if n is None:
            return True
        if n == 2:
            del self.block_refs[block]
        else:
            self.block_refs[block] = n - 1
        return False

    # ---- forking and compacting ----------------------------------------------
    def _copy_blocks(self, src: List[int], dst: List[int]) -> None:
        """Blocks ``src`` to ``dst`` in every layer, K and V, scales included: a launch
        for every 256 of them on the current stream (CPU pools: torch)."""
        if not src:
            return
        if self.block_pool.is_cuda:
            from .. import kernels as K

            with torch.cuda.device(self.block_pool.device):
                K.copy_pages(self.block_pool, src, dst, scales=self.scales)
            return
        pool = self.block_pool.view(torch.uint8)
        pool[:, :, dst] = pool[:, :, src]
        if self.scales is not None:
            self.scales[:, :, dst] = self.scales[:, :, src]

    def fork(self, parent_id: str, child_id: str) -> bool:
        """``child_id`` continues from where ``parent_id`` is (see ``fork_many``)."""
        return self.fork_many([(parent_id, child_id)])

    def fork_many(self, pairs: Sequence[Tuple[str, str]]) -> bool:
        """Give each new request ``child`` the cached tokens of its ``parent``: full blocks
        are shared, a partly filled last block is copied (all pairs' copies together).
        All-or-nothing: False, with nothing changed, when a parent is unknown, a child is
        known or named twice, or the pool has too few free blocks.  Call it between steps:
        the copy is ordered on the current stream."""
        with self._lock:
            children = [c for _, c in pairs]
            if any(p not in self.request_blocks for p, _ in pairs) or \
                    any(c in self.request_blocks for c in children) or \
                    len(set(children)) != len(children):
                return False
            own = [p for p, _ in pairs if self.request_pos[p] < self.block_size]
            if len(own) > len(self.free_blocks):
                return False
            fresh = dict(zip((i for i, (p, _) in enumerate(pairs)
                              if self.request_pos[p] < self.block_size), reversed(self.free_blocks)))
            copies = [(self.request_blocks[pairs[i][0]][-1], b) for i, b in fresh.items()
                      if self.request_pos[pairs[i][0]]]
            self._copy_blocks([s for s, _ in copies], [d for _, d in copies])
            for i, (parent, child) in enumerate(pairs):  # the device work is under way: book it
                table = list(self.request_blocks[parent])
                if i in fresh:
                    table[-1] = self.free_blocks.pop()
                for b in table[:-1] if i in fresh else table:
                    self.block_refs[b] = self.block_refs.get(b, 1) + 1
                self.request_blocks[child] = table
                self.request_pos[child] = self.request_pos[parent]
            return True

    def compact(self) -> int:
        """Move the live blocks into the first ones of the pool (copies on the current
        stream) and hand out the lowest free block first from then on; returns how many
        moved.  Call it between steps: slots reserved before it are no longer valid."""
        with self._lock:
            live = sorted({b for t in self.request_blocks.values() for b in t})
            n = len(live)
            src = [b for b in live if b >= n]
            dst = sorted(set(range(n)) - set(live))
            self._copy_blocks(src, dst)
            moved = dict(zip(src, dst))
            for t in self.request_blocks.values():
                t[:] = [moved.get(b, b) for b in t]
            self.block_refs = {moved.get(b, b): r for b, r in self.block_refs.items()}
            self.free_blocks[:] = range(self.max_num_blocks - 1, n - 1, -1)
            self._pending.clear()
            return len(src)

    def clear(self) -> None:
        with self._lock:
            self.request_blocks.clear()
            self.request_pos.clear()
            self.block_refs.clear()
            self._pending.clear()
            self.free_blocks = list(range(self.max_num_blocks))

    def get_stats(self) -> dict:
        with self._lock:
            used = self.max_num_blocks - len(self.free_blocks)
            return {
                "type": "paged",
                "active_requests": len(self.request_blocks),
                "used_blocks": used,
                "free_blocks": len(self.free_blocks),
                "max_blocks": self.max_num_blocks,
                "block_size": self.block_size,
                "total_tokens": sum(self.get_seq_len(r) for r in self.request_blocks),
                "utilization": used / self.max_num_blocks if self.max_num_blocks else 0,
                "memory_mb": (self.block_pool.numel() * self.block_pool.element_size()
                              + (0 if self.scales is None else self.scales.numel() * 4)) / 2**20,
            }


# Reference class name kept for drop-in callers.
MuPagedCache = PagedKVCache


def create_cache(config, num_layers: int, num_kv_heads: int, head_dim: int, device: str = "cuda",
                 mu_config: Optional[MuConfig] = None, dtype: Optional[torch.dtype] = None):
    """Factory mirroring cache.py:465-515.  Only the paged cache exists here:
    the dense MuKVCache alternative is not on the paged forward path."""
    if not config.use_paged:
        raise NotImplementedError("mu_b200 implements the paged KV cache only (use_paged=True)")
    dtype_map = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32,
                 "float8_e4m3": torch.float8_e4m3fn}
    dt = dtype or dtype_map.get(config.dtype, torch.bfloat16)
    nblocks = config.num_gpu_blocks or config.max_num_blocks
    return PagedKVCache(num_layers, num_kv_heads, head_dim, config.block_size, nblocks, dt, device,
                        mu_config)
