"""Who holds which cache block when sequences share them: forks, copies before a write, release, compaction.  The bookkeeping
is host code; pools on the CPU hold the block numbers, and a fake copy moves them."""
import random

import pytest
import torch

from deltazip_b200.cache import PagedKVCache, RecurrentStateCache
from deltazip_b200.engine import Sequence


class Cache(PagedKVCache):
    """Pools on the CPU; copies are done by indexing."""

    def __init__(self, blocks, block_size=4, window=None, state=None):
        super().__init__(1, blocks, 1, block_size, torch.float32, "cpu", layer_shapes=[(1, 2, 0)], window=window, state=state)
        self.k[0].zero_()
        self.copies = []

    def copy(self, src, dst, rows=None):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        self.copies.append((list(src), list(dst), None if rows is None else list(rows)))
        page = self.k[0].view(self.num_blocks, self.block_size, -1)
        for i, (s, d) in enumerate(zip(src, dst)):
            n = self.block_size if rows is None else rows[i]
            page[d, :n] = page[s, :n]

    def write(self, seq, token):
        """The next token of `seq`, as a decode step does."""
        (slot,) = self.slots(seq.blocks, seq.length, 1)
        self.k[0][slot] = token
        seq.length += 1

    def read(self, seq):
        return [int(self.k[0][s, 0, 0]) for s in self.slots(seq.blocks, 0, seq.length)]

    def consistent(self, seqs):
        held = [0] * self.num_blocks
        for s in seqs:
            for b in s.blocks:
                held[b] += 1
        assert held == self.holders and self.shared == sum(max(0, n - 1) for n in held)
        assert sorted(self.free) == [b for b, n in enumerate(held) if n == 0]


def seq(i, length=0):
    return Sequence(i, 0, length, 0)


def test_fork_shares_and_own_copies_what_is_in_use():
    c = Cache(16)
    a, b = seq(0), seq(1)
    c.open(a, 12)
    for t in range(6):
        c.write(a, 10 + t)
    c.fork([(a, b)])
    b.length = a.length
    c.consistent([a, b])
    assert a.blocks == b.blocks and len(c.free) == 13
    assert c.own([(a, 1), (b, 1)])
    c.consistent([a, b])
    assert a.blocks[0] == b.blocks[0] and a.blocks[1] != b.blocks[1]
    assert c.copies == [([b.blocks[1]], [a.blocks[1]], [2])]         # two tokens of the block; the last holder keeps it
    c.write(a, 1)
    c.write(b, 2)
    assert c.read(a) == [10, 11, 12, 13, 14, 15, 1] and c.read(b) == [10, 11, 12, 13, 14, 15, 2]
    assert not c.own([(a, 1), (b, 1)])
    c.write(a, 3)
    c.write(b, 4)
    assert c.own([(a, 1), (b, 1)]) and c.copies[1] == ([], [], [])   # a shared block nothing is written in yet
    c.close(a)
    c.consistent([b])
    c.close(b)
    c.consistent([])
    assert len(c.free) == 16


def test_a_portion_owns_every_block_it_reaches():
    c = Cache(32)
    a, b, d = seq(0), seq(1), seq(2)
    c.open(a, 20)
    for t in range(7):
        c.write(a, t)
    c.fork([(a, b), (a, d)])
    b.length = d.length = 7
    c.own([(b, 9)])
    c.consistent([a, b, d])
    assert [x == y for x, y in zip(a.blocks, b.blocks)] == [True, False, False, False, True]
    assert c.copies == [([a.blocks[1]], [b.blocks[1]], [3])]


def test_ring_blocks_are_copied_whole():
    c = Cache(16, window=8)
    a, b = seq(0), seq(1)
    c.open(a, 100)
    assert len(a.blocks) == 2
    for t in range(10):
        c.write(a, t)
    c.fork([(a, b)])
    b.length = 10
    c.own([(a, 1), (b, 1)])
    assert c.copies == [([b.blocks[0]], [a.blocks[0]], [4])]
    c.consistent([a, b])


def test_out_of_blocks_changes_nothing():
    c = Cache(3)
    a, b = seq(0), seq(1)
    c.open(a, 12)
    a.length = 6
    c.fork([(a, b)])
    b.length = 6
    was = (list(c.holders), list(a.blocks), list(b.blocks))
    with pytest.raises(RuntimeError):
        c.own([(a, 1), (b, 1)])
    assert was == (c.holders, a.blocks, b.blocks)
    c.consistent([a, b])


def test_release_twice_is_refused():
    c = Cache(4)
    blocks = c.allocate(2)
    c.release(blocks)
    with pytest.raises(RuntimeError):
        c.release(blocks)


def test_random_lives():
    """Forks, writes, closes and compactions in any order: every sequence keeps reading what it wrote."""
    rng = random.Random(4)
    for trial in range(30):
        c = Cache(60)
        live, told, made = [], {}, 0
        for step in range(80):
            what = rng.random()
            if not live or (what < 0.1 and len(live) < 6):
                s = seq(made)
                made += 1
                c.open(s, 20)
                live.append(s)
                told[s.seq_id] = []
            elif what < 0.25 and len(live) < 8:
                parents = rng.sample(live, min(2, len(live)))
                children = [seq(made + i, p.length) for i, p in enumerate(parents)]
                made += len(children)
                c.fork(list(zip(parents, children)))
                for p, s in zip(parents, children):
                    told[s.seq_id] = list(told[p.seq_id])
                live += children
            elif what < 0.35:
                c.close(live.pop(rng.randrange(len(live))))
            elif what < 0.4:
                used = c.compact(live)
                assert sorted(c.free) == list(range(used, 60)) and used == len({b for s in live for b in s.blocks})
            else:
                todo = [s for s in rng.sample(live, rng.randint(1, len(live))) if s.length < 20]
                if sum(c.holders[s.blocks[s.length // 4]] > 1 for s in todo) <= len(c.free):
                    c.own([(s, 1) for s in todo])
                    for s in todo:
                        told[s.seq_id].append(rng.randrange(1000))
                        c.write(s, told[s.seq_id][-1])
            c.consistent(live)
            for s in live:
                assert c.read(s) == told[s.seq_id]


def test_compact_wants_every_holder():
    c = Cache(8)
    a, b = seq(0), seq(1)
    c.open(a, 8)
    c.open(b, 8)
    c.close(a)
    with pytest.raises(ValueError):
        c.compact([])
    was = list(b.blocks)
    assert c.compact([b]) == 2 and sorted(b.blocks) == [0, 1] and c.free == [7, 6, 5, 4, 3, 2]
    assert c.copies == [(sorted(x for x in was if x > 1), [x for x in (0, 1) if x not in was], None)]


def test_copies_are_checked():
    c = PagedKVCache(0, 8, 1, 4, torch.float16, "cpu")
    for bad in (([0], [8]), ([-1], [2]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0], [1, 2]), ([0], [1], [1, 2])):
        with pytest.raises(ValueError):
            c.copy(*bad)
    c.copy([0], [1])
    st = RecurrentStateCache([(1, 2, 3)], 4, "cpu")
    for bad in (([4], [0]), ([0, 1], [2, 2]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            st.copy(*bad)
    for bad in (([0, 1], [0, 2]), ([0, 1], [0]), ([0, 1], [-1, 0])):
        with pytest.raises(ValueError):
            st.reorder(*bad)


def test_states_fork_with_their_sequences():
    class States(RecurrentStateCache):
        def copy(self, src, dst):
            self.log = (src, dst)
    c = Cache(8, state=States([(1, 2, 3)], 3, "cpu"))
    a, b, d = seq(0), seq(1), seq(2)
    c.open(a, 4)
    c.fork([(a, b), (a, d)])
    assert c.state.log == ([a.state_slot] * 2, [b.state_slot, d.state_slot]) and len({a.state_slot, b.state_slot, d.state_slot}) == 3
    with pytest.raises(RuntimeError):
        c.fork([(a, seq(3))])
    c.consistent([a, b, d])
    c.close(b)
    assert c.state.free == [b.state_slot] or b.state_slot == -1


def test_what_one_hypothesis_holds_is_not_shared_when_it_forks():
    """A prompt left with one hypothesis, whose written, partly written and reserved blocks are all its own, forks inside a
    block: only the full blocks both hold count as shared, and both read what they wrote."""
    from deltazip_b200.engine import _Beams
    c = Cache(32)
    root = seq(0)
    c.open(root, 26)
    g = _Beams(0, root)
    for t in range(5):
        c.write(root, t)
    assert g.shared_blocks(4) == 1
    c.write(root, 5)
    child = seq(1, root.length)
    c.fork([(root, child)])
    g.seqs = [root, child]
    assert c.own([(s, 1) for s in g.seqs])
    assert g.shared_blocks(4) == 1
    for step in range(10):
        for i, s in enumerate(g.seqs):
            c.write(s, 100 * (i + 1) + step)
        c.own([(s, 1) for s in g.seqs])
        shared = g.shared_blocks(4)
        assert shared * 4 <= 6 and all(s.blocks[:shared] == root.blocks[:shared] for s in g.seqs)
    assert [c.read(s)[6:] for s in g.seqs] == [[100 * (i + 1) + step for step in range(10)] for i in range(2)]
    c.close(child)
    g.seqs = [root]
    assert g.shared_blocks(4) == 4                    # 16 tokens are written, and blocks behind them reserved
