"""A small decode engine over the delta layers: sequences, the paged KV cache, delta-aware
admission and the per-step device state.  It stands where the reference's scheduler and model
runner stand around the SBMM path (serving/vllm/core/scheduler.py:359-366,528-535: a batch may
hold at most `max_deltas` distinct deltas and is sorted by delta id, :101-104;
serving/vllm/worker/model_runner.py:919-975: set the active deltas and the mapping, run the
model, sample) -- reduced to greedy sampling and to what the throughput configurations need.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, NamedTuple, Optional, Tuple

import torch

from . import ops, registry
from .cache import AttnMeta
from .config import DeltaConfig
from .layers import DeltaMapping
from .models import LRUCacheDeltaModelManager


@dataclass
class Sequence:
    seq_id: int
    delta_id: int                       # 0 = base model
    length: int                         # tokens in the cache so far
    max_new: int
    blocks: List[int] = field(default_factory=list)
    state_slot: int = -1                # recurrent models: slot of this sequence's state
    generated: int = 0
    arrival: float = 0.0
    prompt: Optional[torch.Tensor] = None
    first_token_time: Optional[float] = None


class Hypothesis(NamedTuple):
    """A finished continuation of a beam search."""
    tokens: List[int]
    score: float                        # log-probability / length ** length_penalty


class _Beams:
    """The search for one prompt: its running hypotheses, best first, and what has ended."""

    def __init__(self, number: int, root: Sequence):
        self.number, self.root, self.first_id = number, root, root.seq_id
        self.seqs, self.tokens, self.scores = [root], [[]], [0.0]
        self.common = 0                 # leading cache blocks that all hypotheses hold and have filled
        self.ended: List[Hypothesis] = []

    def end(self, tokens: List[int], score: float, keep: int, penalty: float) -> None:
        self.ended.append(Hypothesis(tokens, score / len(tokens) ** penalty))
        self.ended.sort(key=lambda h: -h.score)
        del self.ended[keep:]

    def decided(self, keep: int, max_new: int, penalty: float) -> bool:
        """Whether no running hypothesis can still pass the worst of `keep` that have ended: its log-probability only
        falls, and a longer continuation is divided by more."""
        if len(self.ended) < keep or not self.scores:
            return not self.scores
        length = max_new if penalty > 0 else len(self.tokens[0]) + 1
        return self.scores[0] / length ** penalty <= self.ended[-1].score

    def shared_blocks(self, block_size: int) -> int:
        """Leading blocks that all hypotheses hold and none will write to again (later ones go on from these)."""
        blocks, full = [s.blocks for s in self.seqs], min(s.length for s in self.seqs) // block_size
        while self.common < full and len({b[self.common] for b in blocks}) == 1:
            self.common += 1
        return self.common


class DecodeEngine:
    """Model + slot manager + sequence cache for one tensor-parallel rank.

    The model is built at random from `cfg` or handed in (`model=`, for a loaded checkpoint).
    Without `delta_config` the base model is served alone.  `max_prefill_tokens` bounds the rows of
    one forward pass for models that can continue a prompt from the cache."""

    def __init__(self, cfg, delta_config: Optional[DeltaConfig], max_seqs: int, kv_blocks: int,
                 block_size: int = 16, device="cuda", dtype=None, seed: int = 0, model=None,
                 max_prefill_tokens: int = 8192):
        self.cfg, self.device, self.block_size = cfg, torch.device(device), block_size
        self.model = model if model is not None else registry.build_model(cfg, device=device, seed=seed, dtype=dtype)
        self.manager = None
        if delta_config is not None:
            if self.model.dtype == torch.float32:
                raise ValueError("deltas are applied to 16-bit activations")
            self.manager = LRUCacheDeltaModelManager(self.model, max_seqs,
                                                     max(max_seqs, 2048, max_prefill_tokens
                                                         if self.model.supports_portions else 0),
                                                     cfg.vocab_size, delta_config, device=device)
        self.cache = self.model.make_cache(kv_blocks, block_size, max_seqs)
        self.max_prefill_tokens = max_prefill_tokens
        self.max_seqs = max_seqs
        self.running: List[Sequence] = []
        self._dirty = True
        self._order: List[int] = []
        self.tokens = None
        self.positions = None
        self.block_tables = None
        self.attn_splits = 0            # 0: chosen per step from the batch (see decode_step)
        self.groups = None              # sequences of the batch that share blocks: (sizes, shared lengths), see beam_search
        self.swap_ins = 0

    # -- batch composition -----------------------------------------------------------
    def admit(self, waiting: List[Sequence]) -> List[Sequence]:
        """Delta-aware admission: sequences join while a batch slot, KV blocks for their whole
        life and a GPU slot for their delta are available.  A delta that is not resident takes a
        free slot or evicts the least recently used delta no running sequence needs.  Returns
        the sequences admitted (their deltas are resident and activated)."""
        admitted = []
        mgr = self.manager
        in_use = {s.delta_id for s in self.running if s.delta_id > 0}
        for seq in list(waiting):
            if len(self.running) + len(admitted) >= self.max_seqs:
                break
            tokens = seq.length + seq.max_new
            if not self.cache.can_open(tokens):
                continue
            d = seq.delta_id
            if d > 0 and mgr is None:
                continue                                        # no deltas are served here
            if d > 0 and d not in mgr._active_deltas:
                if mgr.get_delta(d) is None:
                    continue                                    # unknown delta: not servable
                if len(mgr._active_deltas) + len(mgr._loading) >= mgr.delta_slots and d not in mgr._loading:
                    victim = next((x for x in mgr._active_deltas if x not in in_use), None)
                    if victim is None:
                        continue                                # every slot is needed by the batch
                    mgr.deactivate_delta(victim)
                mgr.activate_delta(d)
            elif d > 0:
                mgr._active_deltas.move_to_end(d)
            in_use.add(d)
            self.cache.open(seq, tokens)
            admitted.append(seq)
            waiting.remove(seq)
        if admitted:
            self.running.extend(admitted)
            self._dirty = True
        return admitted

    def admit_overlapped(self, waiting: List[Sequence], ready=None) -> List[Sequence]:
        """Admission that never makes the compute stream wait for a swap-in: a sequence whose
        delta is not resident triggers a prefetch into a free (or evictable) GPU slot -- the
        upload runs on the copy stream while the batch keeps decoding -- and joins in a later
        round, once the upload's event has completed.  `ready(delta_id) -> bool` reports that
        (default: the event's own query; a tensor-parallel caller passes the agreement of all
        ranks so that every rank admits the same sequences)."""
        mgr = self.manager
        if ready is None:
            def ready(d):
                return mgr._slot_ready[mgr._loading[d]].query()
        admitted = []
        in_use = {s.delta_id for s in self.running if s.delta_id > 0}
        wanted = set()
        for seq in list(waiting):
            if len(self.running) + len(admitted) >= self.max_seqs:
                break
            tokens = seq.length + seq.max_new
            if not self.cache.can_open(tokens):
                continue
            d = seq.delta_id
            if d > 0 and mgr is None:
                continue                                        # no deltas are served here
            if d > 0 and d not in mgr._active_deltas:
                if mgr.get_delta(d) is None:
                    continue
                if d in mgr._loading:
                    if not ready(d):
                        continue
                    mgr.activate_delta(d)              # upload finished: no stall
                else:
                    if d in wanted:
                        continue
                    if len(mgr._active_deltas) + len(mgr._loading) >= mgr.delta_slots:
                        victim = next((x for x in mgr._active_deltas if x not in in_use), None)
                        if victim is None:
                            continue
                        mgr.deactivate_delta(victim)
                    mgr.prefetch_delta(d)
                    self.swap_ins += 1
                    wanted.add(d)
                    continue
            elif d > 0:
                mgr._active_deltas.move_to_end(d)
            in_use.add(d)
            self.cache.open(seq, tokens)
            admitted.append(seq)
            waiting.remove(seq)
        if admitted:
            self.running.extend(admitted)
            self._dirty = True
        return admitted

    def retire(self, seq: Sequence) -> None:
        self.cache.close(seq)
        self.running.remove(seq)
        self._dirty = True

    def compact(self) -> int:
        """Moves the cache blocks in use to the lowest numbers; returns how many there are."""
        used = self.cache.compact(self.running)
        self._dirty = True
        return used

    def _slot_of(self, delta_id: int) -> int:
        return self.manager.delta_index_to_id.index(delta_id) if delta_id > 0 else -1

    def _sort_key(self, seq: Sequence):
        return (self._slot_of(seq.delta_id), seq.seq_id)

    def _set_mapping(self, seqs: List[Sequence], counts: List[int]) -> None:
        if self.manager is not None:
            ids = [s.delta_id for s, n in zip(seqs, counts) for _ in range(n)]
            self.manager.set_delta_mapping(DeltaMapping(ids, [s.delta_id for s in seqs]))

    def _block_tables(self, seqs: List[Sequence]) -> torch.Tensor:
        width = max([len(s.blocks) for s in seqs] + [1])
        tab = torch.zeros((max(len(seqs), 1), width), dtype=torch.int32)
        for i, s in enumerate(seqs):
            tab[i, : len(s.blocks)] = torch.tensor(s.blocks, dtype=torch.int32)
        return tab.to(self.device)

    def _int32(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def _state_slots(self, seqs: List[Sequence]) -> Optional[torch.Tensor]:
        return self._int32([s.state_slot for s in seqs]) if self.cache.state is not None else None

    def _rebuild(self, tokens: Optional[Dict[int, int]] = None) -> None:
        """Device-side state of the running batch, sequences ordered by GPU slot so that the
        token rows reach the SBMM sorted.  `tokens`: seq_id -> next input token."""
        old = {}
        if self.tokens is not None and self._order:
            host = self.tokens.tolist()
            old = {sid: host[i] for i, sid in enumerate(self._order)}
        if tokens:
            old.update(tokens)
        self.running.sort(key=self._sort_key)
        self._order = [s.seq_id for s in self.running]
        dev = self.device
        self.block_tables = self._block_tables(self.running)
        self.positions = torch.tensor([s.length for s in self.running], dtype=torch.int64, device=dev)
        self.tokens = torch.tensor([old.get(s.seq_id, 0) for s in self.running], dtype=torch.int64,
                                   device=dev)
        self.state_slots = self._state_slots(self.running)
        self.q_starts = torch.arange(len(self.running) + 1, dtype=torch.int32, device=dev)
        self._set_mapping(self.running, [1] * len(self.running))
        self._dirty = False

    # -- one decode step ---------------------------------------------------------------
    def _decode_rows(self) -> torch.Tensor:
        """Feeds every running sequence its latest token; returns the hidden states, rows in the batch's order."""
        if self.cache.own([(s, 1) for s in self.running]):
            self._dirty = True
        if self._dirty:
            self._rebuild()
        bs = self.block_size
        pos = self.positions
        # the modulus only matters for windowed models, whose sequences use their blocks as a ring
        blk = torch.gather(self.block_tables, 1, (pos // bs % self.block_tables.shape[1]).unsqueeze(1))
        slot = blk.squeeze(1).to(torch.int64) * bs + pos % bs
        lens = (pos + 1).to(torch.int32)
        # one CTA per (sequence, kv head, split): split the keys when the batch alone would leave
        # most SMs without a CTA
        splits = self.attn_splits or max(1, min(8, 296 // max(1, len(self.running) * self.model.kv_heads)))
        meta = AttnMeta(slot_mapping=slot, block_tables=self.block_tables, seq_lens=lens,
                        splits=splits, q_starts=self.q_starts, ctx_lens=pos.to(torch.int32),
                        state_slots=self.state_slots)
        if self.groups is not None:
            sizes, shared = self.groups
            meta.group_starts = self._int32([0] + torch.tensor(sizes).cumsum(0).tolist())
            meta.shared_lens, meta.max_group, meta.max_shared = self._int32(shared), max(sizes), max(shared)
        h = self.model(self.tokens, pos, self.cache, meta)
        self.positions = pos + 1
        for s in self.running:
            s.length += 1
            s.generated += 1
        return h

    @torch.inference_mode()
    def decode_step(self) -> torch.Tensor:
        """Feeds every running sequence its latest token (position = its cached length), appends
        the new key/value to the cache and samples the next token greedily.  Device work only
        unless the batch composition changed since the last step."""
        self.tokens = self.model.greedy_tokens(self._decode_rows())
        return self.tokens

    # -- given tokens --------------------------------------------------------------------
    def _forward_rows(self, work: List[Tuple[Sequence, List[int]]]) -> torch.Tensor:
        """One forward pass over the next tokens of some sequences; returns their hidden states, rows
        in the order of `work` (which is sorted by GPU slot)."""
        seqs, counts = [s for s, _ in work], [len(t) for _, t in work]
        dev = self.device
        decode = all(n == 1 for n in counts) and (self.model.supports_portions or all(s.length for s in seqs))
        if not decode and not self.model.supports_portions and any(s.length for s in seqs):
            raise ValueError("this model cannot continue a prompt from its cache")
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        meta = AttnMeta(
            slot_mapping=torch.tensor([x for s, n in zip(seqs, counts)
                                       for x in self.cache.slots(s.blocks, s.length, n)],
                                      dtype=torch.int64, device=dev),
            block_tables=self._block_tables(seqs),
            seq_lens=self._int32([s.length + n for s, n in zip(seqs, counts)]),
            prompt_lens=None if decode else counts,
            q_starts=self._int32(starts), ctx_lens=self._int32([s.length for s in seqs]),
            state_slots=self._state_slots(seqs), host_ctx_lens=[s.length for s in seqs])
        toks = torch.tensor([t for _, ts in work for t in ts], dtype=torch.int64).to(dev)
        pos = torch.tensor([s.length + i for s, n in zip(seqs, counts) for i in range(n)], dtype=torch.int64).to(dev)
        self._set_mapping(seqs, counts)
        self._dirty = True                      # the mapping and the lengths are no longer those of a decode step
        h = self.model(toks, pos, self.cache, meta)
        for s, n in zip(seqs, counts):
            s.length += n
        return h

    @torch.inference_mode()
    def extend(self, work: List[Tuple[Sequence, List[int]]]) -> torch.Tensor:
        """Runs the given next tokens of admitted sequences (new prompts, portions of prompts, single
        tokens, in any mixture) from the cache and state that earlier calls left; a sequence that was
        admitted for fewer tokens takes further cache blocks.  Returns the hidden states of all the
        tokens, in the order of `work`.  Models that support it take long work in passes of at most
        `max_prefill_tokens` rows."""
        for s, toks in work:
            self.cache.reserve(s, s.length + len(toks))
        self.cache.own([(s, len(toks)) for s, toks in work])
        order = sorted(range(len(work)), key=lambda i: self._sort_key(work[i][0]))
        limit = self.max_prefill_tokens if self.model.supports_portions else None
        parts: List[List[torch.Tensor]] = [[] for _ in work]
        done = [0] * len(work)
        while True:
            room, batch = limit, []
            for i in order:
                left = len(work[i][1]) - done[i]
                n = left if room is None else min(left, room)
                if n > 0:
                    batch.append((i, n))
                    room = None if room is None else room - n
            if not batch:
                break
            h = self._forward_rows([(work[i][0], list(work[i][1][done[i]:done[i] + n])) for i, n in batch])
            row = 0
            for i, n in batch:
                parts[i].append(h[row:row + n])
                done[i] += n
                row += n
        rows = [p for ps in parts for p in ps]
        return torch.cat(rows) if rows else torch.empty((0, 0), device=self.device)

    @torch.inference_mode()
    def prefill(self, seqs: List[Sequence]) -> None:
        """Runs the prompts of newly admitted sequences (all tokens of all prompts in one pass where
        they fit, rows sorted by GPU slot), fills their cache blocks and leaves their first generated
        token as the next decode input."""
        if not seqs:
            return
        seqs = sorted(seqs, key=self._sort_key)
        for s in seqs:
            s.length = 0
        h = self.extend([(s, s.prompt.tolist()) for s in seqs])
        last = torch.tensor([int(s.prompt.numel()) for s in seqs], device=self.device).cumsum(0) - 1
        nxt = self.model.greedy_tokens(h[last]).tolist()
        first = {s.seq_id: nxt[i] for i, s in enumerate(seqs)}
        for s in seqs:
            s.generated = 1
        self._rebuild(first)

    # -- whole requests ------------------------------------------------------------------
    def generate(self, prompts: List[List[int]], max_new: int, delta_ids: Optional[List[int]] = None,
                 stop_id: Optional[int] = None) -> List[List[int]]:
        """Greedy generation for a list of prompts through admission, prefill and decode steps: sequences
        join as batch slots, cache and deltas allow and leave when they have `max_new` tokens or
        produced `stop_id`."""
        if self.running:
            raise RuntimeError("sequences are already running")
        if max_new < 1 or any(not p for p in prompts):
            raise ValueError("prompts hold at least a token, and at least one token is generated")
        waiting = [Sequence(i, delta_ids[i] if delta_ids else 0, len(p), max_new,
                            prompt=torch.tensor(p, dtype=torch.int64)) for i, p in enumerate(prompts)]
        out: List[List[int]] = [[] for _ in prompts]

        def take(tokens: List[int], order: List[int], fresh) -> None:
            for sid, tok in zip(order, tokens):
                if sid in fresh:
                    out[sid].append(tok)
            for s in list(self.running):
                if s.seq_id in fresh and (s.generated >= max_new or out[s.seq_id][-1] == stop_id):
                    self.retire(s)

        while waiting or self.running:
            admitted = self.admit(waiting)
            if admitted:
                self.prefill(admitted)
                take(self.tokens.tolist(), self._order, {s.seq_id for s in admitted})
            elif not self.running:
                raise RuntimeError("a waiting request fits neither the cache nor the resident deltas")
            if self.running:
                toks = self.decode_step().tolist()
                take(toks, self._order, set(self._order))
        return out

    # -- beam search ---------------------------------------------------------------------
    def _most_blocks(self, prompt: int, max_new: int, beams: int) -> int:
        """Cache blocks that the hypotheses of a prompt hold at most: full blocks of the prompt together, the rest each by
        itself (a ring is written all over)."""
        total = self.cache.blocks_for(prompt + max_new)
        common = prompt // self.block_size if self.cache.window is None else 0
        return common + beams * (total - common)

    @torch.inference_mode()
    def beam_search(self, prompts: List[List[int]], max_new: int, beams: int, delta_ids: Optional[List[int]] = None,
                    stop_id: Optional[int] = None, length_penalty: float = 1.0) -> List[List[Hypothesis]]:
        """The best continuations of each prompt by log-probability / length ** length_penalty that a search with `beams`
        hypotheses finds, best first: of up to `max_new` tokens, or ending in `stop_id`.  Hypotheses share the cache blocks
        of what they have in common, fork by sharing, and copy a block only before they write to it; recurrent states are
        copied.  Prompts join as batch slots (`beams` each), cache and deltas allow."""
        if self.running:
            raise RuntimeError("sequences are already running")
        if max_new < 1 or any(not p for p in prompts):
            raise ValueError("prompts hold at least a token, and at least one token is generated")
        if not getattr(self.model, "whole_vocabulary", True):
            raise ValueError("a beam search needs the whole vocabulary on one rank")
        if not 1 <= beams <= min(self.max_seqs, 64):
            raise ValueError(f"between 1 and {min(self.max_seqs, 64)} hypotheses a prompt")
        waiting = [_Beams(i, Sequence(i * beams, delta_ids[i] if delta_ids else 0, len(p), max_new,
                                      prompt=torch.tensor(p, dtype=torch.int64))) for i, p in enumerate(prompts)]
        need = {g.number: self._most_blocks(g.root.length, max_new, beams) for g in waiting}
        keep = beams if stop_id is None else 2 * beams          # as many again may end here
        out: List[List[Hypothesis]] = [[] for _ in prompts]
        active: List[_Beams] = []
        try:
            while waiting or active:
                fresh = []
                for g in list(waiting):
                    if (len(active) + len(fresh) + 1) * beams > self.max_seqs or \
                            sum(need[x.number] for x in active + fresh + [g]) > self.cache.num_blocks:
                        break
                    if self.admit([g.root]):
                        fresh.append(g)
                        waiting.remove(g)
                if fresh:
                    for g in fresh:
                        g.root.length = 0
                    h = self.extend([(g.root, g.root.prompt.tolist()) for g in fresh])
                    last = torch.tensor([g.root.length for g in fresh], device=self.device).cumsum(0) - 1
                    active += fresh
                    self._select(fresh, h[last], keep, beams, max_new, stop_id, length_penalty, active, out)
                elif not active:
                    raise RuntimeError("a waiting request fits neither the cache nor the resident deltas")
                if active:
                    self._rebuild_beams(active)
                    self._select(active, self._decode_rows(), keep, beams, max_new, stop_id, length_penalty, active, out)
        finally:
            self.groups = None
            for s in list(self.running):
                self.retire(s)
        return out

    def _rebuild_beams(self, active: List[_Beams]) -> None:
        """The batch of all hypotheses, each prompt's side by side, and what they share."""
        self.cache.own([(s, 1) for g in active for s in g.seqs])
        self._order, tokens = [], {}
        for g in active:
            for i, s in enumerate(g.seqs):
                s.seq_id = g.first_id + i
                tokens[s.seq_id] = g.tokens[i][-1]
        self._rebuild(tokens)
        active.sort(key=lambda g: self._sort_key(g.seqs[0]))
        self.groups = ([len(g.seqs) for g in active],
                       [g.shared_blocks(self.block_size) * self.block_size if self.cache.window is None else 0 for g in active])

    def _select(self, groups: List[_Beams], hidden: torch.Tensor, keep: int, beams: int, max_new: int, stop_id: Optional[int],
                penalty: float, active: List[_Beams], out: List[List[Hypothesis]]) -> None:
        """Continues the hypotheses of `groups` (their hidden states in this order) by their best next tokens; groups that
        are through leave `active` with their results."""
        starts = [0]
        for g in groups:
            starts.append(starts[-1] + len(g.seqs))
        scores = torch.tensor([x for g in groups for x in g.scores], dtype=torch.float32).to(self.device)
        best = ops.beam_select(self.model.beam_logits(hidden), scores, self._int32(starts), keep)
        best_scores, rows, tokens = (t.tolist() for t in best)
        forks = []
        for i, g in enumerate(list(groups)):
            nxt = []
            for rank, (score, row, token) in enumerate(zip(best_scores[i], rows[i], tokens[i])):
                if score == float("-inf") or len(nxt) == beams:
                    break
                parent = row - starts[i]
                if token != stop_id:
                    nxt.append((parent, g.tokens[parent] + [token], score))
                elif rank < beams:
                    g.end(g.tokens[parent] + [token], score, beams, penalty)
            if nxt and len(nxt[0][1]) == max_new:
                for _, toks, score in nxt:
                    g.end(toks, score, beams, penalty)
                nxt = []
            old, g.tokens, g.scores = g.seqs, [t for _, t, _ in nxt], [x for _, _, x in nxt]
            through = g.decided(beams, max_new, penalty)
            heirs = set() if through else {p for p, _, _ in nxt}
            for p, s in enumerate(old):
                if p not in heirs:
                    self.retire(s)
            if through:
                out[g.number] = g.ended
                active.remove(g)
                continue
            g.seqs, taken = [], set()
            for p, _, _ in nxt:                                 # the first heir takes the sequence itself
                if p in taken:
                    child = Sequence(-1, old[p].delta_id, old[p].length, max_new, generated=old[p].generated)
                    forks.append((old[p], child))
                    g.seqs.append(child)
                else:
                    taken.add(p)
                    g.seqs.append(old[p])
        self.cache.fork(forks)
        self.running.extend(child for _, child in forks)
        self._dirty = True
