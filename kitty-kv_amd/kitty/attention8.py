"""Layers whose keys and values stay in 8 bits: the cache of all their sequences
and an attention module with ``KittyPagedAttention``'s ``forward``.

No counterpart in the reference, whose only cache is the 2-bit one.  It is for
layers that 2 bits cost too much (often the first and the last of a model):
``KittyAttentionFactory.from_config(..., eight_bit_layers=(0, 31))`` builds them
next to the 2-bit ones.  At head_dim 128 a token takes 256 bytes a KV head against
76 in 2 bits and 512 in 16.

A page holds ``q_buffer_size`` tokens (16, 32, 64, 128 or 256) of one sequence and
stands at the same place in every layer's pools, so one block table serves all
layers; a layer's pools hold ``max_seq_len`` tokens of every slot, or
``pool_pages_override`` pages if that is less.
Tokens are quantised as they are written (``kernels.cache8``), there are no 16-bit
sinks or windows, and a chunk of any length attends over everything its sequence
holds, itself included.  No step waits for the GPU: lengths live on the device and
in a host copy, and only new pages send their ids over.  (For that host copy a step
that adds tokens is not captured into a graph; the calls of ``Cache8`` are.)
"""
from __future__ import annotations

import heapq
import math
from typing import Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
import torch.nn as nn

from .config import KittyConfig
from .kernels.cache8 import Cache8
from .kernels.ops import stage_i32


class KittyCache8:
    """8-bit pools of `num_layers` layers and the sequences in them.

    It counts their tokens and pages: what `layers[i]` writes or evicts beside it, it
    does not know of."""

    def __init__(self, config: KittyConfig, num_layers: Optional[int] = None) -> None:
        self.config = config
        L = config.num_layers if num_layers is None else int(num_layers)
        H, G, D, n = config.num_kv_heads, config.q_buffer_size, config.head_dim, config.max_batch_size
        self.max_pages_per_seq = -(-config.max_seq_len // G)
        P = _layer_pages(config, n * self.max_pages_per_seq)
        self.dtype = torch.float16 if config.dtype == "float16" else torch.bfloat16
        self.layers: List[Cache8] = [Cache8.empty(P, H, D, G, device=config.device) for _ in range(L)]
        self.device = self.layers[0].device if L else torch.device(config.device)
        # a row per slot, and one of no tokens for sequences that hold none
        self.block_table = torch.zeros(n + 1, self.max_pages_per_seq, dtype=torch.int32, device=self.device)
        self.lens = torch.zeros(L, n + 1, dtype=torch.int32, device=self.device)     # tokens by layer and slot
        self._held = np.zeros((L, n + 1), np.int64)                                  # the same on the host
        self._pages: List[List[int]] = [[] for _ in range(n)]
        self._fresh, self._freed, self._num_pages = 0, [], P
        self._slot_of: Dict[int, int] = {}
        self._free_slots = list(range(n))
        self._slots_dev: Dict[tuple, torch.Tensor] = {}

    # -------------------------------------------------------------- bookkeeping
    def slot(self, seq_id: int) -> int:
        """Slot of a sequence, assigned (lowest free) on first use."""
        s = self._slot_of.get(seq_id)
        if s is None:
            if not self._free_slots:
                raise RuntimeError(f"all {len(self._pages)} sequence slots are in use; "
                                   "raise KittyConfig.max_batch_size or reset finished sequences")
            s = self._slot_of[seq_id] = heapq.heappop(self._free_slots)
        return s

    def tokens(self, seq_id: int, layer: int = 0) -> int:
        """Tokens a sequence holds in a layer."""
        return int(self._held[layer, self._slot_of[seq_id]]) if seq_id in self._slot_of else 0

    @property
    def pages_free(self) -> int:
        return self._num_pages - self._fresh + len(self._freed)

    def _i32(self, values: Sequence[int]) -> torch.Tensor:
        if self.device.type == "cpu":
            return torch.tensor(list(values), dtype=torch.int32)
        return stage_i32(np.asarray(values, np.int32), self.device)

    def _join(self, layer: int, seq_ids: Sequence[int], tokens: int) -> Tuple[List[int], List[int], List[int]]:
        """Slots of the sequences, with pages for `tokens` more tokens of each, all or
        nothing; also which sequences are new and how many pages each slot got."""
        new = [i for i in seq_ids if i not in self._slot_of]
        if len(new) > len(self._free_slots):
            raise RuntimeError(f"all {len(self._pages)} sequence slots are in use; "
                               "raise KittyConfig.max_batch_size or reset finished sequences")
        taken = dict(zip(new, heapq.nsmallest(len(new), self._free_slots)))
        slots = [self._slot_of.get(i, taken.get(i)) for i in seq_ids]
        G = self.config.q_buffer_size
        need = [max(0, -(-(int(self._held[layer, s]) + tokens) // G) - len(self._pages[s])) for s in slots]
        for s, n in zip(slots, need):
            if len(self._pages[s]) + n > self.max_pages_per_seq:
                raise RuntimeError(f"a sequence exceeds max_seq_len={self.config.max_seq_len}")
        if sum(need) > self.pages_free:
            raise RuntimeError(f"KV Cache page pool exhausted! {self.pages_free} free pages, {sum(need)} needed.")
        for i in new:
            self.slot(i)
        for s, n in zip(slots, need):
            if n == 0:
                continue
            ids = []
            for _ in range(n):
                if self._freed:
                    ids.append(heapq.heappop(self._freed))
                else:
                    ids.append(self._fresh)
                    self._fresh += 1
            at = len(self._pages[s])
            self._pages[s] += ids
            self.block_table[s, at:at + n].copy_(self._i32(ids))
        return slots, new, need

    def _leave(self, slots: Sequence[int], new: Sequence[int], got: Sequence[int]) -> None:
        """Takes a _join back."""
        for s, n in zip(slots, got):
            for _ in range(n):
                heapq.heappush(self._freed, self._pages[s].pop())
        for i in new:
            heapq.heappush(self._free_slots, self._slot_of.pop(i))

    def reset_sequence(self, seq_id: int) -> None:
        """Drops a sequence: its pages and its slot are free again."""
        s = self._slot_of.pop(seq_id, None)
        if s is None:
            return
        for p in self._pages[s]:
            heapq.heappush(self._freed, p)
        self._pages[s] = []
        self._held[:, s] = 0
        self.lens[:, s].zero_()
        heapq.heappush(self._free_slots, s)

    # -------------------------------------------------------------------- calls
    def _slots(self, seq_ids: Sequence[int]) -> List[int]:
        """Slots of a batch to read; sequences that hold nothing take none."""
        if len(set(seq_ids)) != len(seq_ids):
            raise ValueError("a sequence appears twice in one batch")
        return [self._slot_of.get(i, len(self._pages)) for i in seq_ids]

    def _rows(self, layer: int, slots: Sequence[int]):
        """Block table and lengths of the slots, and the slots on the device where they are no run."""
        s0 = slots[0] if slots else 0
        if slots == list(range(s0, s0 + len(slots))):
            return self.block_table[s0:s0 + len(slots)], self.lens[layer, s0:s0 + len(slots)], None
        key = tuple(slots)
        idx = self._slots_dev.get(key)
        if idx is None:
            if len(self._slots_dev) >= 64:
                self._slots_dev.clear()
            idx = self._slots_dev[key] = self._i32(slots).long()
        return self.block_table[idx], self.lens[layer][idx], idx

    def push(self, layer: int, keys: torch.Tensor, values: torch.Tensor, seq_ids: Sequence[int]) -> None:
        """T tokens for each of B sequences: keys / values (B, H, T, D).  A call that is
        refused leaves slots, pages and tokens as they were."""
        if keys.shape[0] != len(seq_ids):
            raise ValueError(f"{len(seq_ids)} sequence ids for a batch of {keys.shape[0]}")
        self._slots(seq_ids)
        if keys.shape[0] == 0 or keys.shape[2] == 0:
            return
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("KittyCache8 counts its tokens on the host, so its steps cannot be captured: "
                               "capture the calls of kitty.kernels.Cache8")
        slots, new, got = self._join(layer, seq_ids, keys.shape[2])
        try:
            table, lens, idx = self._rows(layer, slots)
            self.layers[layer].write(keys.to(self.device), values.to(self.device), table, lens)
        except Exception:
            self._leave(slots, new, got)
            raise
        if idx is None:
            lens.add_(keys.shape[2])
        else:
            self.lens[layer].index_add_(0, idx, torch.full_like(lens, keys.shape[2]))
        self._held[layer, slots] += keys.shape[2]

    def attend(self, layer: int, q: torch.Tensor, seq_ids: Sequence[int], sm_scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of the last T tokens of each sequence, q (B, Hq, T, D); zeros
        for a sequence that holds nothing."""
        slots = self._slots(seq_ids)
        table, lens, _ = self._rows(layer, slots)
        longest = int(self._held[layer, slots].max(initial=0))
        return self.layers[layer].attend(q, table, lens, sm_scale=sm_scale, max_tokens=_bucket(longest))

    def read(self, layer: int, seq_ids: Sequence[int], dtype: Optional[torch.dtype] = None):
        """(keys, values) of the sequences, (B, H, longest, D), zeros behind the shorter
        ones; a sequence that was never pushed, or was reset, holds nothing."""
        slots = self._slots(seq_ids)
        table, lens, _ = self._rows(layer, slots)
        return self.layers[layer].read(table, lens, int(self._held[layer, slots].max(initial=0)), dtype=dtype or self.dtype)


def _layer_pages(config: KittyConfig, most: int) -> int:
    """Pages of an 8-bit layer whose slots can name `most`.  pool_pages_override sizes the
    pool that the 2-bit layers share, often for all of them together: here it is a bound.
    Without it, max_pages (it leaves room for the sinks, which are tokens like others here, out)."""
    if config.pool_pages_override is None:
        return max(config.pool_pages, most)
    return min(config.pool_pages, most)


def _bucket(tokens: int) -> int:
    """A length rounded up to a power of two, so that calls of growing sequences share their checks."""
    return 1 << max(tokens - 1, 0).bit_length()


class KittyPagedAttention8(nn.Module):
    """``KittyPagedAttention``'s constructor order and ``forward`` over a ``KittyCache8``."""

    def __init__(self, config: KittyConfig, num_q_heads: int, cache: KittyCache8, layer: int) -> None:
        super().__init__()
        if num_q_heads <= 0 or num_q_heads % config.num_kv_heads:      # or its first call would push, and then raise
            raise ValueError(f"num_q_heads must be a positive multiple of {config.num_kv_heads}")
        self.config = config
        self.num_q_heads = num_q_heads
        self.num_kv_heads = config.num_kv_heads
        self.head_dim = config.head_dim
        self.cache = cache
        self.layer = layer
        self.scale = 1.0 / math.sqrt(config.head_dim)

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                seq_id: Union[int, Sequence[int]] = 0, attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q (B, Hq, T, D), k and v (B, Hkv, T, D): the tokens join the cache, and each
        attends over what its sequence holds up to itself; (B, Hq, T, D) in q's type.
        attention_mask is not read, as in ``KittyPagedAttention``: sequences of unequal
        lengths are told apart by their ids, and a padded prompt goes in without its padding.
        There is no backward: call under torch.no_grad()."""
        B, nqh, T, D = q.shape
        assert nqh == self.num_q_heads
        assert D == self.head_dim
        ids = [seq_id + b for b in range(B)] if isinstance(seq_id, int) else [int(s) for s in seq_id]
        if len(ids) != B:
            raise ValueError(f"{len(ids)} sequence ids for a batch of {B}")
        if B == 0 or T == 0:
            return torch.empty_like(q)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            raise RuntimeError("the 8-bit cache has no backward: call under torch.no_grad()")
        x = q.to(self.cache.device)
        if x.dtype not in (torch.float16, torch.bfloat16):
            x = x.to(self.cache.dtype)
        self.cache.push(self.layer, k, v, ids)
        return self.cache.attend(self.layer, x, ids, self.scale).to(q.device, q.dtype)
