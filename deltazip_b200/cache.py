"""What a sequence leaves behind between steps: paged key/value pools and recurrent state slots,
and the description of a batch that the model's mixers read them through (role of the reference's
block manager + cache engine, serving/vllm/core/block_manager.py,
serving/vllm/worker/cache_engine.py, reduced to what a single process needs)."""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import torch

from . import ops


def _copy(handle: "ops.PagePools", device, src: Sequence[int], dst: Sequence[int], rows: Optional[Sequence[int]] = None) -> None:
    """copy_pages of pages given as numbers on the host; more than a launch takes go in several (none of them is then both
    source and destination)."""
    if not src or handle.table is None:
        return
    most = ops.copy_pages_max_pairs()
    index = torch.tensor([list(src), list(dst)] + ([list(rows)] if rows is not None else []), dtype=torch.int32).to(device)
    for i in range(0, len(src), most):
        part = [t[i:i + most] for t in index]
        ops.copy_pages(handle, part[0], part[1], part[2] if rows is not None else None)


def _check_pages(what: str, pages: Sequence[int], count: int, distinct: bool = False) -> None:
    if any(not 0 <= p < count for p in pages) or (distinct and len(set(pages)) != len(pages)):
        raise ValueError(f"{what} are {'different ' if distinct else ''}numbers from 0 to {count - 1}")


class RecurrentStateCache:
    """Per recurrent layer run the 32-bit pools S [slots, heads, dim, vdim] and, where the run normalises
    (`normalised`, default: all do), n [slots, heads, dim] and m [slots, heads]; a sequence owns one
    slot number, the same in every pool.  Slots are handed out as they are: a sequence without context
    starts from zero without reading its slot."""

    def __init__(self, shapes: Sequence[Tuple[int, int, int]], slots: int, device="cuda",
                 normalised: Optional[Sequence[bool]] = None):
        f32 = dict(dtype=torch.float32, device=device)
        with_n = [True] * len(shapes) if normalised is None else list(normalised)
        self.S = [torch.zeros((slots, h, d, v), **f32) for h, d, v in shapes]
        self.n = [torch.zeros((slots, h, d), **f32) if w else None for (h, d, _), w in zip(shapes, with_n)]
        self.m = [torch.zeros((slots, h), **f32) if w else None for (h, _, _), w in zip(shapes, with_n)]
        self.free: List[int] = list(range(slots - 1, -1, -1))
        self.slots, self.device = slots, device
        self._pools: Optional[ops.PagePools] = None

    def allocate(self) -> int:
        if not self.free:
            raise RuntimeError("out of recurrent state slots")
        return self.free.pop()

    def release(self, slot: int) -> None:
        self.free.append(slot)

    def copy(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """The states in slots `dst` become those that slots `src` held before, in every run, all at once."""
        _check_pages("slots", src, self.slots)
        _check_pages("slots that are written", dst, self.slots, distinct=True)
        if len(src) != len(dst):
            raise ValueError("a source for every destination")
        if self._pools is None:
            self._pools = ops.PagePools([t for t in self.S + self.n + self.m if t is not None])
        if len(src) > ops.copy_pages_max_pairs() and set(src) & set(dst):
            raise ValueError(f"at most {ops.copy_pages_max_pairs()} slots that follow one another at once")
        _copy(self._pools, self.device, src, dst)

    def reorder(self, slots: Sequence[int], parents: Sequence[int]) -> None:
        """Sequence i of those in `slots` goes on from the state of sequence parents[i] (a number among them)."""
        _check_pages("parents", parents, len(slots))
        if len(slots) != len(parents):
            raise ValueError("a parent for every slot")
        moved = [(slots[p], s) for s, p in zip(slots, parents) if slots[p] != s]
        self.copy([a for a, _ in moved], [b for _, b in moved])


class PagedKVCache:
    """Per-layer K and V pools of `num_blocks` blocks of `block_size` tokens, [slots, kv_heads,
    head size] each, with a free list.  `layer_shapes` gives (kv_heads, key size, value size) per
    layer run where layers differ (default: `num_layers` times (kv_heads, 128, 128)); a run that caches
    one row per token for all heads has one key head and value size 0.

    `window`: the largest number of tokens any layer looks back (itself included).  A sequence then
    owns at most ceil(window / block_size) blocks and uses them as a ring: token position t lives in
    block number (t / block_size) modulo the blocks it owns.  `state` holds the recurrent layers'
    slots, where the model has any.

    Sequences may share blocks (`fork`).  A block goes back to the free list when the last of them gives it up, and `own`
    gives a sequence a copy of a shared block before it writes to it."""

    def __init__(self, num_layers: int, num_blocks: int, kv_heads: int, block_size: int = 16,
                 dtype=torch.float16, device="cuda",
                 layer_shapes: Optional[Sequence[Tuple[int, int, int]]] = None,
                 window: Optional[int] = None, state: Optional[RecurrentStateCache] = None):
        self.block_size, self.num_blocks, self.kv_heads = block_size, num_blocks, kv_heads
        shapes = [(kv_heads, 128, 128)] * num_layers if layer_shapes is None else list(layer_shapes)
        rows = num_blocks * block_size
        self.k = [torch.empty((rows, h, dk), dtype=dtype, device=device) for h, dk, _ in shapes]
        self.v = [torch.empty((rows, h, dv), dtype=dtype, device=device) for h, _, dv in shapes]
        self.window = window
        self.state = state
        self.free: List[int] = list(range(num_blocks - 1, -1, -1))
        self.device = device
        self.holders: List[int] = [0] * num_blocks              # sequences that hold a block
        self.shared = 0                                         # holders beyond the first, over all blocks
        self._pools: Optional[ops.PagePools] = None

    def blocks_for(self, tokens: int) -> int:
        """Blocks a sequence of `tokens` tokens holds at most."""
        if self.window is not None:
            tokens = min(tokens, self.window)
        return (tokens + self.block_size - 1) // self.block_size

    def allocate(self, n_blocks: int) -> List[int]:
        if n_blocks > len(self.free):
            raise RuntimeError("out of KV cache blocks")
        blocks = [self.free.pop() for _ in range(n_blocks)]
        for b in blocks:
            self.holders[b] = 1
        return blocks

    def release(self, blocks: Sequence[int]) -> None:
        """Gives up one holder's claim on each of `blocks`."""
        for b in blocks:
            if self.holders[b] < 1:
                raise RuntimeError(f"cache block {b} is not in use")
            self.holders[b] -= 1
            if self.holders[b]:
                self.shared -= 1
            else:
                self.free.append(b)

    def slots(self, blocks: Sequence[int], start: int, count: int) -> List[int]:
        """Cache slots of token positions [start, start + count) of a sequence owning `blocks`.  Where
        the ring comes round inside the range only its last tokens get a slot (-1: not kept)."""
        bs = self.block_size
        if self.window is None:
            return [blocks[p // bs] * bs + p % bs for p in range(start, start + count)]
        n = len(blocks)
        keep = start + count - n * bs
        return [blocks[p // bs % n] * bs + p % bs if p >= keep else -1 for p in range(start, start + count)]

    # -- whole sequences ---------------------------------------------------------------
    def can_open(self, tokens: int) -> bool:
        return self.blocks_for(tokens) <= len(self.free) and (self.state is None or bool(self.state.free))

    def open(self, seq, tokens: int) -> None:
        """Gives `seq` (an object with `blocks` and `state_slot`) what it needs for `tokens` tokens."""
        seq.blocks = self.allocate(self.blocks_for(tokens))
        if self.state is not None:
            seq.state_slot = self.state.allocate()

    def reserve(self, seq, tokens: int) -> None:
        """Gives an open `seq` the blocks it still lacks for `tokens` tokens.  (A ring has all it will ever
        have: its positions are counted modulo its blocks.)"""
        if self.window is None and len(seq.blocks) < self.blocks_for(tokens):
            seq.blocks = seq.blocks + self.allocate(self.blocks_for(tokens) - len(seq.blocks))

    def close(self, seq) -> None:
        self.release(seq.blocks)
        seq.blocks = []
        if self.state is not None and seq.state_slot >= 0:
            self.state.release(seq.state_slot)
            seq.state_slot = -1

    # -- shared blocks -----------------------------------------------------------------
    def fork(self, pairs: Sequence[Tuple[object, object]]) -> None:
        """For (parent, child) pairs the child goes on from what the parent has in the cache: it holds the same blocks and,
        with recurrent layers, a copy of the state in a slot of its own (one launch for all pairs)."""
        if self.state is not None and len(pairs) > len(self.state.free):
            raise RuntimeError("out of recurrent state slots")
        for parent, child in pairs:
            child.blocks = list(parent.blocks)
            for b in child.blocks:
                self.holders[b] += 1
            self.shared += len(child.blocks)
            if self.state is not None:
                child.state_slot = self.state.allocate()
        if self.state is not None:
            self.state.copy([p.state_slot for p, _ in pairs], [c.state_slot for _, c in pairs])

    def own(self, work: Sequence[Tuple[object, int]]) -> bool:
        """Before (sequence, count) write `count` tokens from position sequence.length on: the blocks these go to become the
        sequence's own, a shared one as a copy of what it holds of the tokens before (one launch for all).  Returns whether
        any sequence's blocks changed."""
        if not self.shared:
            return False
        bs, todo = self.block_size, []
        for seq, count in work:
            seen = set()
            for at in range(seq.length // bs, (seq.length + count - 1) // bs + 1 if count > 0 else 0):
                # a ring's block still holds tokens of the last round behind the one that is written
                i, rows = (at, max(0, seq.length - at * bs)) if self.window is None else (at % len(seq.blocks), bs)
                if self.holders[seq.blocks[i]] > 1 and i not in seen:
                    seen.add(i)
                    todo.append((seq, i, rows))
        left, new = {}, []
        for seq, i, _ in todo:                                  # who comes last keeps the block
            b = seq.blocks[i]
            left[b] = left.get(b, self.holders[b]) - 1
            new.append(left[b] > 0)
        if sum(new) > len(self.free):
            raise RuntimeError("out of KV cache blocks")
        src, dst, kept = [], [], []
        for (seq, i, rows), fresh in zip(todo, new):
            if not fresh:
                continue
            (b,) = self.allocate(1)
            if rows:
                src.append(seq.blocks[i])
                dst.append(b)
                kept.append(rows)
            self.release([seq.blocks[i]])
            seq.blocks = seq.blocks[:i] + [b] + seq.blocks[i + 1:]
        self.copy(src, dst, kept)
        return any(new)

    def copy(self, src: Sequence[int], dst: Sequence[int], rows: Optional[Sequence[int]] = None) -> None:
        """Copies the first `rows` tokens (default: all) of blocks `src` to blocks `dst` in every run; no block is both."""
        _check_pages("blocks", src, self.num_blocks)
        _check_pages("blocks that are written", dst, self.num_blocks, distinct=True)
        if len(src) != len(dst) or (rows is not None and len(rows) != len(src)) or set(src) & set(dst):
            raise ValueError("a source for every destination, and none of them a destination")
        if not src or not any(t.numel() for t in self.k + self.v):
            return
        if self._pools is None:
            self._pools = ops.PagePools(self.k + self.v, self.block_size)
        _copy(self._pools, self.device, src, dst, rows)

    def compact(self, seqs: Sequence[object]) -> int:
        """Moves the blocks in use to the lowest numbers, so that all behind them are free; `seqs`: every sequence that
        holds any.  Returns how many there are."""
        held: dict = {}
        for seq in seqs:
            for b in seq.blocks:
                held[b] = held.get(b, 0) + 1
        if any(held.get(b, 0) != n for b, n in enumerate(self.holders)):
            raise ValueError("all sequences that hold blocks have to be given")
        used = len(held)
        high = sorted(b for b in held if b >= used)
        move = dict(zip(high, (b for b in range(used) if b not in held)))
        self.copy(list(move), list(move.values()))
        for a, b in move.items():
            self.holders[b], self.holders[a] = self.holders[a], 0
        for seq in seqs:
            seq.blocks = [move.get(b, b) for b in seq.blocks]
        self.free = list(range(self.num_blocks - 1, used - 1, -1))
        return used


@dataclass
class AttnMeta:
    """How the sequence mixers run in one forward pass; rows are in (sequence, position) order.

    Decode (`prompt_lens` is None): one row per sequence; `block_tables` [B, max_blocks] int32 and
    `seq_lens` [B] int32 (cached length including the current token).
    Prompt portions: `prompt_lens`, the row count of each sequence.

    Models that continue prompts from a cache also read `q_starts` [B + 1] int32 (first row of every
    sequence), `ctx_lens` [B] int32 (tokens before the first row; `host_ctx_lens` the same as numbers, for
    prompt portions) and, with recurrent layers, `state_slots` [B] int32.  `shared` keeps what the layers
    of one pass derive from all this.

    Where sequences share cache blocks, a decode step may say so: sequences group_starts[g] ... group_starts[g + 1] - 1
    have their first shared_lens[g] tokens in common, `max_group` and `max_shared` being the largest of both."""
    slot_mapping: Optional[torch.Tensor] = None          # int64 [M] cache slot per token, -1 = none
    block_tables: Optional[torch.Tensor] = None
    seq_lens: Optional[torch.Tensor] = None
    prompt_lens: Optional[List[int]] = None
    splits: int = 1
    q_starts: Optional[torch.Tensor] = None
    ctx_lens: Optional[torch.Tensor] = None
    state_slots: Optional[torch.Tensor] = None
    host_ctx_lens: Optional[List[int]] = None
    positions: Optional[torch.Tensor] = None             # int64 [M], set by models whose mixers read them
    shared: dict = field(default_factory=dict)
    group_starts: Optional[torch.Tensor] = None          # int32 [G + 1]
    shared_lens: Optional[torch.Tensor] = None           # int32 [G]
    max_group: int = 0
    max_shared: int = 0

    @property
    def decode(self) -> bool:
        return self.prompt_lens is None

    @property
    def max_query(self) -> int:
        return 1 if self.prompt_lens is None else max(self.prompt_lens)
