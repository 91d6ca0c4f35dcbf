"""State caches of the GDN layers, in the layout the kernels read.

Replaces ``LinearAttentionCache`` (``cache/linear_attention_cache.py:7-88`` of
yuyifanbupt/myvllm) with the same constructor arguments, slot allocator and
zero-on-free semantics, and these corrections:

* the recurrent (SSM) cache holds ``num_v_heads`` heads, the heads the
  kernels index (the reference sizes it with ``num_k_heads``, ``:37-45``);
* the recurrent state is fp32 (``state_dtype``), whatever the activations'
  dtype (the reference uses the model dtype for both caches, ``:27``);
* the conv cache has its own dtype (``conv_dtype``, default the model dtype);
* freeing a slot zeroes it in every layer with one device fill per cache
  (the reference issues two fills per layer, ``:83-85``).

Layouts: conv cache ``(layers, slots, W-1, D)`` with ``D = 2 K Hk + V Hv``
channels q | k | v, token-major, oldest row first; recurrent cache
``(layers, slots, Hv, K, V)`` with ``[K][V]`` contiguous per head.  A layer's
views (``layer(l)``) are what ``causal_conv1d_fn`` / ``causal_conv1d_update`` /
``chunk_gated_delta_rule`` / ``recurrent_gated_delta_rule`` /
``gated_delta_net_decode_step`` take, indexed by the allocated slot ids.

Beside it stands the paged cache of the attention layers (:class:`PagedKVCache`),
whose sequences share pages after a fork, and the copy that both fork with
(:func:`cache_copy`).
"""
from __future__ import annotations

from array import array
from collections import deque
from collections.abc import Sequence

import torch

from . import _lib


def cache_copy(caches: torch.Tensor | Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Copies blocks inside caches, in place: in every layer of every cache
    (layers, blocks, ...), block ``dst[i]`` becomes block ``src[i]``; the step behind a
    fork or a compaction.  Any element type; the caches have one number of blocks,
    the elements of a block lie side by side, and no two blocks overlap (an expanded view).

    ``src`` and ``dst`` are on the host (lists, CPU tensors or arrays of whole numbers),
    where a cache's allocator has them: they travel with the launch, and a captured
    call replays its own.  The places are distinct and none of them is a source, ids are
    inside the caches: checked before anything is copied."""
    caches = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    if not caches:
        raise ValueError("no caches to copy in")
    if _lib.copy_caches(caches, src, dst):
        return
    _lib.require_device(*caches)
    pairs = _pairs(src, dst)
    rows = []
    for t in caches:
        if t.dim() < 3:
            raise ValueError(f"caches are (layers, blocks, ...), got {tuple(t.shape)}")
        if t.shape[1] != caches[0].shape[1]:
            raise ValueError("caches of one call have one number of blocks")
        if t.numel() and not t[0, 0].is_contiguous():
            raise ValueError("the elements of a block must lie side by side")
        t = t.detach().flatten(2) if t.numel() else t.detach().reshape(t.shape[0], t.shape[1], 0)
        rows.append(t if t.dtype in _lib.DTYPE_CODES else t.view(torch.uint8))
    if pairs.shape[1] == 0:
        return
    for i in range(0, len(rows), 4):
        part = rows[i: i + 4]
        _lib.call("cache_copy", *part, *[None] * (4 - len(part)), pairs)


def _pairs(src, dst) -> torch.Tensor:
    """(2, n) int32 on the host."""
    if isinstance(src, torch.Tensor) and src.is_cuda or isinstance(dst, torch.Tensor) and dst.is_cuda:
        raise ValueError("src and dst are on the host")
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} sources for {len(dst)} places")
    try:
        ids = array("i", src)
        ids.extend(array("i", dst))
    except OverflowError:
        raise ValueError("block ids outside the caches") from None
    return torch.frombuffer(ids, dtype=torch.int32).view(2, -1) if ids else torch.empty(2, 0, dtype=torch.int32)


class LinearAttentionCache:
    def __init__(
        self,
        layer_cnt: int,
        max_seq_cnt: int,
        conv_kernel_size: int,
        k_head_dim: int,
        v_head_dim: int,
        num_k_heads: int,
        num_v_heads: int,
        dtype: torch.dtype,
        device: torch.device,
        state_dtype: torch.dtype = torch.float32,
        conv_dtype: torch.dtype | None = None,
    ) -> None:
        if num_k_heads <= 0 or num_v_heads % num_k_heads != 0:
            raise ValueError("num_v_heads must be a positive multiple of num_k_heads")
        self.layer_cnt = layer_cnt
        self.max_seq_cnt = max_seq_cnt
        self.conv_kernel_size = conv_kernel_size
        self.k_head_dim = k_head_dim
        self.v_head_dim = v_head_dim
        self.num_k_heads = num_k_heads
        self.num_v_heads = num_v_heads
        self.dtype = dtype
        self.state_dtype = state_dtype
        self.conv_dtype = conv_dtype or dtype
        self.device = device
        self.conv_dim = 2 * k_head_dim * num_k_heads + v_head_dim * num_v_heads
        self.conv_cache = torch.zeros(
            layer_cnt, max_seq_cnt, conv_kernel_size - 1, self.conv_dim, dtype=self.conv_dtype, device=device
        )
        self.recurrent_cache = torch.zeros(
            layer_cnt, max_seq_cnt, num_v_heads, k_head_dim, v_head_dim, dtype=state_dtype, device=device
        )
        self.free_slot_ids: deque[int] = deque(range(max_seq_cnt))
        self.used_slot_ids: set[int] = set()

    @staticmethod
    def bytes_per_seq(
        layer_cnt: int,
        conv_kernel_size: int,
        k_head_dim: int,
        v_head_dim: int,
        num_k_heads: int,
        num_v_heads: int,
        dtype: torch.dtype,
        state_dtype: torch.dtype = torch.float32,
        conv_dtype: torch.dtype | None = None,
    ) -> int:
        """Cache bytes one sequence slot takes over all layers."""
        conv_dtype = conv_dtype or dtype
        conv = layer_cnt * (conv_kernel_size - 1) * (2 * k_head_dim * num_k_heads + v_head_dim * num_v_heads)
        recurrent = layer_cnt * num_v_heads * k_head_dim * v_head_dim
        return conv * conv_dtype.itemsize + recurrent * state_dtype.itemsize

    def layer(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(conv_state (slots, W-1, D), recurrent_state (slots, Hv, K, V)) views of one layer."""
        return self.conv_cache[layer_idx], self.recurrent_cache[layer_idx]

    def can_allocate(self) -> bool:
        return len(self.free_slot_ids) > 0

    def allocate(self) -> int:
        if not self.free_slot_ids:
            raise RuntimeError("no free cache slot")
        slot_id = self.free_slot_ids.popleft()
        self.used_slot_ids.add(slot_id)
        return slot_id

    def fork(self, slot_id: int) -> int:
        """A new slot that holds slot_id's states, in every layer."""
        return self.fork_many([slot_id])[0]

    def fork_many(self, slot_ids) -> list[int]:
        """One new slot for each of slot_ids (which may repeat), in one copy."""
        slot_ids = [int(s) for s in slot_ids]
        for s in slot_ids:
            if s not in self.used_slot_ids:
                raise ValueError(f"slot {s} is not allocated")
        if len(slot_ids) > len(self.free_slot_ids):
            raise RuntimeError("no free cache slot")
        new = [self.free_slot_ids[i] for i in range(len(slot_ids))]
        cache_copy([self.conv_cache, self.recurrent_cache], slot_ids, new)
        return [self.allocate() for _ in new]

    def deallocate(self, slot_id: int) -> None:
        self.deallocate_many([slot_id])

    def deallocate_many(self, slot_ids) -> None:
        """Free slots (zeroed in every layer; later frees are reused first, as
        one ``deallocate`` after another in the reference)."""
        slot_ids = [int(s) for s in slot_ids]
        for s in slot_ids:
            if s not in self.used_slot_ids:
                raise ValueError(f"slot {s} is not allocated")
        if len(set(slot_ids)) != len(slot_ids):
            raise ValueError("slot ids repeat")
        if slot_ids:
            idx = torch.tensor(slot_ids, dtype=torch.long, device=self.device)
            self.conv_cache.index_fill_(1, idx, 0)
            self.recurrent_cache.index_fill_(1, idx, 0)
        for s in slot_ids:
            self.used_slot_ids.remove(s)
            self.free_slot_ids.appendleft(s)


class PagedKVCache:
    """Paged keys and values of the attention layers, with the tables of the
    sequences in them (no counterpart in the reference, which has the paged ops
    but no cache for them).

    Tensors: ``k_cache``, ``v_cache`` (layers, blocks, block_size, heads, head_dim) in
    ``dtype``; with ``bits=4`` uint8 codes (head_dim / 2) and ``k_scales``,
    ``v_scales`` (layers, blocks, heads, head_dim / 32, block_size), as
    ``paged_kv_append`` writes them.  :meth:`layer` gives a layer's.

    A sequence is an id with its blocks and its length.  A fork shares the blocks of its
    sequence; whoever first extends a shared, partly filled one gets a copy of it.
    """

    def __init__(
        self,
        layer_cnt: int,
        block_cnt: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device,
        bits: int = 16,
    ) -> None:
        if bits not in (4, 16):
            raise ValueError("caches are held in 16 or 4 bits")
        if bits == 4 and (block_size % 16 or head_dim % 32):
            raise ValueError("caches held in 4 bits have blocks of a multiple of 16 slots and heads of 32 dims")
        self.layer_cnt = layer_cnt
        self.block_cnt = block_cnt
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.bits = bits
        self.device = device
        shape = (layer_cnt, block_cnt, block_size, num_kv_heads)
        row, kind = (head_dim, dtype) if bits == 16 else (head_dim // 2, torch.uint8)
        self.k_cache, self.v_cache = (torch.zeros(*shape, row, dtype=kind, device=device) for _ in range(2))
        self.k_scales = self.v_scales = None
        if bits == 4:
            shape = (layer_cnt, block_cnt, num_kv_heads, head_dim // 32, block_size)
            self.k_scales, self.v_scales = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        self.free_block_ids: deque[int] = deque(range(block_cnt))
        self.holders = [0] * block_cnt  # sequences that hold each block
        self.blocks: dict[int, list[int]] = {}
        self.lengths: dict[int, int] = {}
        self._next_id = 0

    @staticmethod
    def bytes_per_block(layer_cnt: int, block_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype,
                        bits: int = 16) -> int:
        """Cache bytes one block takes over all layers, keys and values."""
        row = head_dim * dtype.itemsize if bits == 16 else head_dim // 2 + head_dim // 32
        return 2 * layer_cnt * block_size * num_kv_heads * row

    def layer(self, layer_idx: int):
        """(k_cache, v_cache, k_scales, v_scales) of one layer; the scales are None in 16 bits."""
        return tuple(None if t is None else t[layer_idx]
                     for t in (self.k_cache, self.v_cache, self.k_scales, self.v_scales))

    def _tensors(self) -> list[torch.Tensor]:
        return [t for t in (self.k_cache, self.v_cache, self.k_scales, self.v_scales) if t is not None]

    def _check(self, seq_ids) -> None:
        for s in seq_ids:
            if s not in self.blocks:
                raise ValueError(f"sequence {s} is not in the cache")
        if len(set(seq_ids)) != len(seq_ids):
            raise ValueError("sequence ids repeat")

    def _take(self) -> int:
        b = self.free_block_ids.popleft()
        self.holders[b] = 1
        return b

    def allocate(self) -> int:
        """A new, empty sequence's id."""
        s = self._next_id
        self._next_id += 1
        self.blocks[s], self.lengths[s] = [], 0
        return s

    def extend(self, seq_ids, counts) -> None:
        """Room for ``counts[i]`` more tokens of each sequence: new blocks, and copies
        of the shared blocks that they would be written to, all in one.  Raises with
        nothing changed when the free blocks are too few.  ``paged_kv_append`` takes
        the tables and lengths (:meth:`tables`) from here."""
        seq_ids, counts = [int(s) for s in seq_ids], [int(n) for n in counts]
        self._check(seq_ids)
        if len(counts) != len(seq_ids) or min(counts, default=0) < 0:
            raise ValueError("one count of new tokens for each sequence, none below 0")
        need, shared = 0, []
        held: dict[int, int] = {}
        for s, n in zip(seq_ids, counts):
            have, size = self.blocks[s], self.lengths[s]
            need += -(-(size + n) // self.block_size) - len(have)
            if n and size % self.block_size:
                last = have[-1]
                if held.setdefault(last, self.holders[last]) > 1:  # (its last holder writes to it where it lies)
                    held[last] -= 1
                    shared.append(s)
        if need + len(shared) > len(self.free_block_ids):
            raise RuntimeError("no free cache block")
        if shared:
            src = [self.blocks[s][-1] for s in shared]
            dst = [self.free_block_ids[i] for i in range(len(shared))]
            cache_copy(self._tensors(), src, dst)
            for s, b in zip(shared, src):
                self.holders[b] -= 1
                self.blocks[s][-1] = self._take()
        for s, n in zip(seq_ids, counts):
            self.lengths[s] += n
            while len(self.blocks[s]) * self.block_size < self.lengths[s]:
                self.blocks[s].append(self._take())

    def fork(self, seq_id: int) -> int:
        """A new sequence with seq_id's tokens, which shares its blocks."""
        self._check([seq_id])
        new = self.allocate()
        self.blocks[new], self.lengths[new] = list(self.blocks[seq_id]), self.lengths[seq_id]
        for b in self.blocks[new]:
            self.holders[b] += 1
        return new

    def free(self, seq_ids) -> None:
        """Ends sequences; blocks that nobody holds any more are free (the most recently
        freed is taken first, as the slots of the state cache are)."""
        seq_ids = [int(s) for s in seq_ids]
        self._check(seq_ids)
        for s in seq_ids:
            for b in self.blocks.pop(s):
                self.holders[b] -= 1
                if self.holders[b] == 0:
                    self.free_block_ids.appendleft(b)
            del self.lengths[s]

    def compact(self) -> int:
        """Moves the blocks in use to the cache's front, in one copy, and returns how many
        moved.  Tables made before are stale."""
        used = self.block_cnt - len(self.free_block_ids)
        src = [b for b in range(used, self.block_cnt) if self.holders[b]]
        dst = [b for b in range(used) if not self.holders[b]]
        if src:
            cache_copy(self._tensors(), src, dst)
        to = dict(zip(src, dst))
        for blocks in self.blocks.values():
            blocks[:] = [to.get(b, b) for b in blocks]
        for a, b in to.items():
            self.holders[b], self.holders[a] = self.holders[a], 0
        self.free_block_ids = deque(range(used, self.block_cnt))
        return len(src)

    def tables(self, seq_ids) -> tuple[torch.Tensor, torch.Tensor]:
        """(block_tables (N, most blocks), context_lens (N,)), int32, as the paged ops
        take them; entries past a sequence's blocks are -1.  Made anew on the host by
        each call, once a step for all layers: 2.7 ms for 64 sequences of U[1024, 8192]
        tokens in blocks of 16, 19 for 256 of U[512, 16384]."""
        seq_ids = [int(s) for s in seq_ids]
        for s in seq_ids:
            if s not in self.blocks:
                raise ValueError(f"sequence {s} is not in the cache")
        cols = max([len(self.blocks[s]) for s in seq_ids], default=0) or 1
        rows = [self.blocks[s] + [-1] * (cols - len(self.blocks[s])) for s in seq_ids]
        return (torch.tensor(rows, dtype=torch.int32).view(len(seq_ids), cols).to(self.device),
                torch.tensor([self.lengths[s] for s in seq_ids], dtype=torch.int32).to(self.device))
