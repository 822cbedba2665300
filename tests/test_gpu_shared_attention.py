"""Decode attention of sequences that share their first pages, against softmax attention in 64 bits: groups from one
sequence to more rows than a CTA takes, lengths around its 16-key tiles, four warps and parts, pages that end inside a
tile, empty groups and sequences, and what is refused.

Tolerance: scores, sums and weights are 32-bit, so what is left is the output's rounding, at most half a unit in the
last place: 2^-11 (fp16) or 2^-8 (bf16) of every element; twice that for the relative 2-norm of a sequence."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float16: 2 * 2.0 ** -11, torch.bfloat16: 2 * 2.0 ** -8}
SCALE = 128 ** -0.5


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """Groups of sequences; `shared`: keys of every group, `fresh`: further keys of every sequence."""

    def __init__(self, sizes, shared, fresh, heads, kvh, dtype, block=16, seed=0, extra_pages=0):
        g, rng = torch.Generator("cuda").manual_seed(seed), random.Random(seed)
        rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
        self.heads, self.kvh, self.block, self.dtype, self.sizes, self.shared = heads, kvh, block, dtype, sizes, shared
        self.group = [i for i, n in enumerate(sizes) for _ in range(n)]
        self.starts = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
        n = len(self.group)
        self.lens = [shared[i] + f for i, f in zip(self.group, fresh)]
        full = [s // block for s in shared]                        # pages that are common; the rest of a prompt is copied
        wide = max([-(-x // block) for x in self.lens] + [1]) + extra_pages
        pages = sum(full) + n * wide
        order = rng.sample(range(pages), pages)
        common = [[order.pop() for _ in range(f)] for f in full]
        self.tables = [(common[i] + [order.pop() for _ in range(wide)])[:wide] for i in self.group]
        self.k, self.v = 2 * rnd(pages * block, kvh, 128), rnd(pages * block, kvh, 128)
        self.qkv = rnd(n, (heads + 2 * kvh) * 128)
        for s, i in enumerate(self.group):                         # a partly filled page holds the same keys for all
            for t in range(full[i] * block, shared[i]):
                a, b = self.slot(self.starts[i], t), self.slot(s, t)
                self.k[b], self.v[b] = self.k[a], self.v[a]

    def slot(self, s, t):
        return self.tables[s][t // self.block] * self.block + t % self.block

    def run(self, shared=None, most=None, longest=None, **kw):
        from deltazip_b200 import ops
        shared = self.shared if shared is None else shared
        return ops.shared_attention_decode(
            kw.pop("qkv", self.qkv), self.k, self.v, i32(self.tables), i32(self.lens), i32(self.starts), i32(shared),
            max(self.sizes) if most is None else most, max(shared) if longest is None else longest, self.heads, self.kvh, self.block,
            SCALE, **kw)

    def want(self, s):
        n, rep = self.lens[s], self.heads // self.kvh
        at = torch.tensor([self.slot(s, t) for t in range(n)], dtype=torch.long, device="cuda")
        k, v = (t[at].double().repeat_interleave(rep, 1) for t in (self.k, self.v))
        q = self.qkv[s, :self.heads * 128].view(self.heads, 128).double()
        p = (torch.einsum("hd,khd->hk", q, k) * SCALE).softmax(1)
        return torch.einsum("hk,khd->hd", p, v).reshape(-1)

    def check(self, out):
        assert torch.isfinite(out).all()
        for s in range(len(self.group)):
            if self.lens[s] == 0:
                assert not out[s].any()
                continue
            want = self.want(s)
            err = (out[s].double() - want).norm() / want.norm()
            assert err <= TOL[self.dtype], (s, float(err))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kvh", [(4, 4), (8, 1), (12, 3), (16, 1), (5, 5)])
@pytest.mark.parametrize("sizes", [[1], [4], [3, 1, 8], [9, 2]])
def test_groups(sizes, heads, kvh, dtype):
    rng = random.Random(heads + len(sizes))
    shared = [rng.choice([1, 15, 16, 17, 64, 65, 130, 700]) for _ in sizes]
    fresh = [rng.choice([0, 1, 16, 33, 200]) for _ in range(sum(sizes))]
    Batch(sizes, shared, fresh, heads, kvh, dtype, seed=heads).check(Batch(sizes, shared, fresh, heads, kvh, dtype, seed=heads).run())


@pytest.mark.parametrize("size,heads,kvh", [(16, 2, 2), (17, 1, 1), (33, 2, 2), (70, 1, 1), (12, 8, 1), (5, 16, 1), (9, 14, 2)])
def test_rows_of_a_group(size, heads, kvh):
    """Rows that fill one, two and four warps, and several CTAs."""
    b = Batch([size, 2], [300, 40], [5] * (size + 2), heads, kvh, torch.bfloat16, seed=size)
    b.check(b.run())


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1030])
@pytest.mark.parametrize("shared", [0.0, 0.5, 1.0])
def test_lengths(length, shared):
    n = int(length * shared)
    b = Batch([3, 2], [n, max(0, n - 1)], [length - n] * 5, 4, 2, torch.float16, seed=length)
    b.check(b.run())


@pytest.mark.parametrize("block", [1, 3, 7, 24, 32, 100])
def test_page_sizes(block):
    b = Batch([4, 3], [210, 90], [3, 50, 1, 0, 7, 8, 9], 8, 4, torch.bfloat16, block=block, seed=block)
    b.check(b.run())


def test_many_parts():
    """Few columns and long sequences: shared and own keys in many parts each."""
    b = Batch([2], [20000], [9000, 12000], 2, 1, torch.float16, seed=3)
    b.check(b.run())
    b = Batch([1, 1], [0, 0], [9000, 12000], 2, 1, torch.float16, seed=4)
    b.check(b.run())


def test_wide_tables():
    """Parts are counted by the tables' width, of which short sequences fill little."""
    b = Batch([4, 2], [20, 300], [0, 1, 70, 3, 5, 6], 8, 8, torch.float16, seed=5, extra_pages=900)
    b.check(b.run())


def test_sequences_that_do_not_share():
    """Without shared keys, without groups, beyond the largest group, beyond the longest shared length."""
    from deltazip_b200 import ops
    b = Batch([5, 3], [128, 64], [9, 80, 1, 2, 0, 30, 31, 32], 8, 2, torch.float16, seed=6)
    full = b.run()
    b.check(full)
    for kw in (dict(shared=[0, 0]), dict(shared=[-5, 0], longest=0), dict(most=2), dict(most=0), dict(most=1, longest=70), dict(longest=17),
               dict(most=100, longest=10 ** 6)):
        b.check(b.run(**kw))
    none = ops.shared_attention_decode(b.qkv, b.k, b.v, i32(b.tables), i32(b.lens), i32([]), i32([]), 0, 0, b.heads, b.kvh, b.block, SCALE)
    b.check(none)
    some = ops.shared_attention_decode(b.qkv, b.k, b.v, i32(b.tables), i32(b.lens), i32([1, 4]), i32([128]), 3, 128, b.heads, b.kvh,
                                       b.block, SCALE)
    b.check(some)


def test_short_and_empty_sequences():
    """A sequence shorter than its group's shared length reads its own pages -- also the group's first, of which nothing
    may be left -- and one without keys gets zeros."""
    b = Batch([4, 2, 0, 1], [100, 50, 30, 0], [5, 6, 7, 8, 1, 2, 0], 4, 4, torch.bfloat16, seed=7)
    for lens in ([0, 106, 107, 108, 51, 52, 0], [105, 40, 0, 108, 0, 0, 0], [99, 100, 101, 1, 49, 50, 0]):
        b.lens = lens
        keep = b.tables[0]
        if lens[0] == 0:
            b.tables[0] = [0] * len(keep)
        b.check(b.run())
        b.tables[0] = keep


def test_rows_with_a_stride():
    b = Batch([3, 2], [70, 20], [5] * 5, 8, 4, torch.float16, seed=8)
    wide = torch.randn((5, b.qkv.shape[1] + 24), device="cuda").half()
    wide[:, 8:8 + b.qkv.shape[1]] = b.qkv
    got = b.run(qkv=wide[:, 8:8 + b.qkv.shape[1]])
    assert torch.equal(got, b.run())
    out = torch.full_like(got, 7)
    assert b.run(out=out) is out and torch.equal(out, got)


def test_pages_outside_the_cache_are_not_read():
    """Entries behind a sequence's keys may be anything; entries of keys that are wrong read some row of the cache."""
    b = Batch([3, 2], [64, 32], [5, 6, 7, 8, 9], 4, 4, torch.float16, seed=9, extra_pages=3)
    want = b.run()
    for i, n in enumerate(b.lens):
        for j in range(-(-n // 16), len(b.tables[i])):
            b.tables[i][j] = (-1, 2 ** 31 - 1, -2 ** 31)[j % 3]
    assert torch.equal(b.run(), want)
    b.tables[1][b.lens[1] // 16] = 2 ** 31 - 1
    b.tables[3][0] = -7
    assert torch.isfinite(b.run()).all()


def test_weights_keep_32_bits():
    """bf16, four keys a sequence whose products with the weights cancel down to 2^-16 of themselves, so that the output's
    own rounding is out of the way.  Error allowed against the sum of absolute products: 2^-19.5, from two units of the
    exponential and three 32-bit sums (2^-21); a weight of two 16-bit parts is off by up to 2^-18."""
    from deltazip_b200 import ops
    n, heads, dtype = 64, 8, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn((n, 1, 128), generator=g, device="cuda").to(dtype)
    k = torch.randn((n * 16, 1, 128), generator=g, device="cuda").to(dtype)
    v = (1 + torch.rand((n, 16, 128), generator=g, device="cuda")).to(dtype)
    w = torch.einsum("nd,nkd->nk", q[:, 0].double(), k.view(n, 16, 128)[:, :4].double()).mul(SCALE).softmax(1)
    for key in (2, 3):                             # each takes away what the keys before it leave
        v[:, key] = (-(w[:, :key, None] * v[:, :key].double()).sum(1) / w[:, key, None]).to(dtype)
    qkv = torch.cat([q.expand(n, heads, 128).reshape(n, -1), torch.zeros((n, 256), device="cuda", dtype=dtype)], 1).contiguous()
    parts = w[:, :, None] * v[:, :4].double()
    for shared in (0, 3, 4):                       # all keys its own, joined from two parts, all shared
        out = ops.shared_attention_decode(qkv, k, v.reshape(-1, 1, 128), i32([[i] for i in range(n)]), i32([4] * n),
                                          i32(list(range(n + 1))), i32([shared] * n), 1, shared, heads, 1, 16, SCALE)
        err = (out.view(n, heads, 128).double() - parts.sum(1)[:, None]).abs() / parts.abs().sum(1)[:, None]
        assert float(err.max()) <= 2.0 ** -19.5, (shared, float(err.max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("key", [0, 5, 69, 70, 75])
def test_infinities_among_the_values(key, dtype):
    """An infinite component of a value gives that infinity, and leaves the other components alone; values behind a
    sequence's end do not count."""
    b = Batch([3], [70], [6, 6, 6], 4, 2, dtype, seed=key)
    b.k *= 0.02
    for s in range(3):
        b.v[b.slot(s, key), :, 7], b.v[b.slot(s, key), :, 12] = float("inf"), float("-inf")
    out = b.run()
    for s in range(3):
        want = b.want(s)
        bad = torch.isinf(want)
        assert int(bad.sum()) == 2 * b.heads and torch.equal(out[s].double()[bad], want[bad])
        err = (out[s].double()[~bad] - want[~bad]).norm() / want[~bad].norm()
        assert err <= TOL[dtype]


def test_nan_behind_the_end():
    """Rows of the cache that no sequence holds may be anything."""
    b = Batch([3, 2], [70, 33], [6, 9, 12, 1, 0], 4, 4, torch.float16, seed=11)
    want = b.run()
    used = {b.slot(s, t) for s in range(5) for t in range(b.lens[s])}
    free = torch.tensor([r for r in range(b.k.shape[0]) if r not in used], device="cuda")
    b.k[free], b.v[free] = float("nan"), float("nan")
    assert torch.equal(b.run(), want)


def test_same_as_reading_by_itself():
    from deltazip_b200 import ops
    b = Batch([6, 2], [512, 100], [40] * 8, 32, 8, torch.float16, seed=12)
    got = b.run()
    alone = ops.paged_attention_decode(b.qkv, b.k, b.v, i32(b.tables), i32(b.lens), 32, 8, 16, SCALE)
    assert float((got.double() - alone.double()).abs().max()) <= 2 * 2.0 ** -11 * float(alone.abs().max())


def test_same_bits_again_and_in_graphs():
    """On a side stream; two captured graphs replayed in turn, the lengths read when they run."""
    from deltazip_b200 import ops
    b = Batch([4, 3], [200, 90], [30] * 7, 8, 2, torch.float16, seed=13)
    want = b.run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    args = [b.qkv, b.k, b.v, i32(b.tables), i32(b.lens), i32(b.starts), i32(b.shared)]
    call = lambda: ops.shared_attention_decode(*args, 4, 200, 8, 2, 16, SCALE)
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(call(), want)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(call())
        graphs.append(g)
    graphs[0].replay()
    torch.cuda.synchronize()
    b.lens = [n - 3 for n in b.lens]
    args[4].copy_(i32(b.lens))
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    b.check(outs[1])


def test_refusals():
    from deltazip_b200 import ops
    from deltazip_b200._lib import DeltaZipError
    b = Batch([2, 1], [20, 3], [5] * 3, 8, 4, torch.float16, seed=14)
    base = dict(qkv=b.qkv, k_cache=b.k, v_cache=b.v, block_tables=i32(b.tables), seq_lens=i32(b.lens), group_starts=i32(b.starts),
                shared_lens=i32(b.shared), max_group=2, max_shared=20, q_heads=8, kv_heads=4, block_size=16, scale=SCALE)
    ops.shared_attention_decode(**base)
    for bad in (dict(max_group=-1), dict(max_shared=-1), dict(block_size=0), dict(q_heads=7), dict(qkv=b.qkv[:, 4:])):
        with pytest.raises((DeltaZipError, ValueError)):
            ops.shared_attention_decode(**{**base, **bad})
    for bad in (dict(seq_lens=i32(b.lens).long()), dict(seq_lens=i32(b.lens[:2])), dict(block_tables=i32(b.tables).t()),
                dict(group_starts=i32(b.starts[:-1])), dict(k_cache=b.k.float()), dict(kv_heads=2), dict(v_cache=b.v[:-16]),
                dict(out=b.qkv), dict(qkv=b.qkv.cpu()), dict(qkv=b.qkv.float())):
        with pytest.raises(ValueError):
            ops.shared_attention_decode(**{**base, **bad})
    wide = Batch([1], [20], [5], 17, 1, torch.float16, seed=15)
    with pytest.raises(DeltaZipError):
        wide.run()
    empty = ops.shared_attention_decode(b.qkv[:0], b.k, b.v, i32(b.tables)[:0], i32([]), i32([]), i32([]), 0, 0, 8, 4, 16, SCALE)
    assert empty.shape == (0, 1024)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,heads,kvh", [(5, 8, 2), (9, 8, 1), (40, 4, 1)])
@pytest.mark.parametrize("key", [0, 63, 64, 141, 149, 155])
def test_infinities_among_the_values_of_many_rows(key, size, heads, kvh, dtype):
    """The same with more rows than eight, sixteen and sixty-four, over three tiles of 64 keys."""
    b = Batch([size, 1], [150, 20], [6] * (size + 1), heads, kvh, dtype, seed=key)
    b.k *= 0.02
    for s in range(size):
        b.v[b.slot(s, key), :, 7], b.v[b.slot(s, key), :, 12] = float("inf"), float("-inf")
    out = b.run()
    for s in range(size):
        want = b.want(s)
        bad = torch.isinf(want)
        assert int(bad.sum()) == 2 * heads and torch.equal(out[s].double()[bad], want[bad])
        err = (out[s].double()[~bad] - want[~bad]).norm() / want[~bad].norm()
        assert err <= TOL[dtype]


@pytest.mark.parametrize("block", [16, 32, 5])
@pytest.mark.parametrize("size,heads,kvh", [(3, 4, 4), (4, 8, 2), (9, 8, 1), (33, 8, 2)])
def test_nan_behind_the_end_of_many_rows(size, heads, kvh, block):
    """Shared lengths that end inside a tile, a box and a page, with NaN in every row of the cache that is not held."""
    shared = [70, 1, 64, 129, 177]
    b = Batch([size] * 5, shared, [i % 20 for i in range(5 * size)], heads, kvh, torch.bfloat16, block=block, seed=size)
    want = b.run()
    b.check(want)
    used = {b.slot(s, t) for s in range(5 * size) for t in range(b.lens[s])}
    free = torch.tensor([r for r in range(b.k.shape[0]) if r not in used], device="cuda")
    b.k[free], b.v[free] = float("nan"), float("nan")
    assert torch.equal(b.run(), want)


@pytest.mark.parametrize("size,heads,kvh", [(3, 2, 2), (5, 8, 2), (9, 8, 1)])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-3, 5.0])
def test_scales(scale, size, heads, kvh):
    from deltazip_b200 import ops
    b = Batch([size, 2], [200, 30], [9] * (size + 2), heads, kvh, torch.float16, seed=3)
    out = ops.shared_attention_decode(b.qkv, b.k, b.v, i32(b.tables), i32(b.lens), i32(b.starts), i32(b.shared), size, 200, heads, kvh,
                                      16, scale)
    global SCALE
    was, SCALE = SCALE, scale
    try:
        b.check(out)
    finally:
        SCALE = was


@pytest.mark.parametrize("sizes", [[9], [12, 3, 16], [16] * 40])
def test_parts_of_every_length(sizes):
    """Groups of more than 16 rows whose parts have one, two and many tiles of 64 keys; a CTA takes several parts."""
    for longest in (1, 64, 65, 128, 700, 5000):
        rng = random.Random(longest)
        shared = [rng.randint(1, longest) for _ in sizes]
        if len(sizes) > 3:
            shared = [min(n, 300) for n in shared]
        b = Batch(sizes, shared, [rng.randint(0, 5) for _ in range(sum(sizes))], 8, 2, torch.float16, seed=longest)
        b.check(b.run())


def test_large_scores_move_the_maximum():
    """Scores that rise along the keys, by more than a step of the running maximum from tile to tile."""
    for size, heads, kvh in ((2, 2, 2), (4, 8, 2), (9, 8, 1)):
        b = Batch([size], [900], [40] * size, heads, kvh, torch.bfloat16, seed=size)
        for s in range(size):
            at = torch.tensor([b.slot(s, t) for t in range(b.lens[s])], device="cuda")
            b.k[at] = (b.k[at].float() * 0.05 + torch.linspace(0, 6, len(at), device="cuda")[:, None, None] *
                       b.qkv[0, :128].float().sign()[None, None]).to(torch.bfloat16)
        b.check(b.run())


@pytest.fixture
def bound_far_above(monkeypatch):
    """A bound on the shared keys far above the ones there are: groups of many rows stay on tensor memory."""
    from deltazip_b200 import ops
    real = ops.shared_attention_decode

    def call(qkv, k, v, tables, lens, starts, shared, most, longest, *rest, **kw):
        return real(qkv, k, v, tables, lens, starts, shared, most, max(longest, 2000), *rest, **kw)
    monkeypatch.setattr(ops, "shared_attention_decode", call)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,heads,kvh", [(5, 8, 2), (9, 8, 1), (40, 4, 1)])
@pytest.mark.parametrize("key", [0, 63, 64, 141, 149, 155])
def test_infinities_in_short_parts_of_tensor_memory(bound_far_above, key, size, heads, kvh, dtype):
    test_infinities_among_the_values_of_many_rows(key, size, heads, kvh, dtype)


@pytest.mark.parametrize("block", [16, 32, 5])
@pytest.mark.parametrize("size,heads,kvh", [(3, 4, 4), (4, 8, 2), (9, 8, 1), (33, 8, 2)])
def test_nan_behind_short_parts_of_tensor_memory(bound_far_above, size, heads, kvh, block):
    test_nan_behind_the_end_of_many_rows(size, heads, kvh, block)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kvh", [(8, 1), (12, 3), (16, 1)])
@pytest.mark.parametrize("sizes", [[4], [3, 1, 8], [9, 2]])
def test_short_parts_in_tensor_memory(bound_far_above, sizes, heads, kvh, dtype):
    test_groups(sizes, heads, kvh, dtype)


@pytest.mark.parametrize("sizes", [[9], [12, 3, 16], [16] * 40])
def test_parts_of_every_length_in_tensor_memory(bound_far_above, sizes):
    test_parts_of_every_length(sizes)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-3, 5.0])
def test_scales_in_tensor_memory(bound_far_above, scale):
    test_scales(scale, 9, 8, 1)


@pytest.mark.parametrize("keys", [511, 512, 513])
@pytest.mark.parametrize("size,heads,kvh", [(5, 8, 2), (9, 8, 1), (20, 2, 2)])
def test_lengths_at_which_the_form_changes(keys, size, heads, kvh):
    b = Batch([size, 2], [keys, 40], [5] * (size + 2), heads, kvh, torch.bfloat16, seed=keys)
    b.check(b.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("groups,size,rep,kvh,own", [(37, 4, 8, 4, False), (222, 2, 8, 8, False), (222, 1, 1, 8, False), (222, 1, 1, 8, True)])
def test_sums_over_long_spans(groups, size, rep, kvh, own, dtype):
    """65536 keys in one part, in tensor memory, on warps with sixteen rows and on warps with few, whose output the last two
    keys cancel, so that its own rounding is out of the way.  Allowed against the sum of absolute products: at most 384
    products of 16 keys go into one accumulator (half of 4096 keys, or 2048, in three parts), an addition loses up to
    2^-22 of a sum that grows evenly to half of the absolute sum -- 384 * 2^-22 / 4 = 2^-15.4 -- and all else, the scores of
    the last two keys above all, stays below 2^-17: 2^-14.9 together.  (The losses have one sign: over all 65536 keys they
    come to between 2^-13 and 2^-11.)"""
    from deltazip_b200 import ops
    n, seqs = 65536, groups * size
    g = torch.Generator("cuda").manual_seed(groups + size)
    q = torch.randn((kvh, 128), generator=g, device="cuda").to(dtype)
    k = torch.randn((n, kvh, 128), generator=g, device="cuda").to(dtype)
    v = (1 + torch.rand((n, kvh, 128), generator=g, device="cuda")).to(dtype)
    k[-2:] = q                                     # weights of the size of all the others together
    w = (torch.einsum("hd,nhd->hn", q.double(), k.double()) * SCALE).softmax(1)
    for j in (n - 2, n - 1):                       # each takes away what the keys before it leave
        v[j] = (-torch.einsum("hn,nhd->hd", w[:, :j], v[:j].double()) / w[:, j, None]).to(dtype)
    heads = kvh * rep
    qkv = torch.cat([q.repeat_interleave(rep, 0).reshape(-1), torch.zeros(2 * kvh * 128, device="cuda", dtype=dtype)])
    shared = [0 if own else n] * groups
    out = ops.shared_attention_decode(qkv.repeat(seqs, 1), k, v, i32([list(range(n // 16))]).repeat(seqs, 1), i32([n] * seqs),
                                      i32(list(range(0, seqs + 1, size))), i32(shared), size, max(shared), heads, kvh, 16, SCALE)
    assert torch.equal(out, out[:1].expand_as(out))
    want, parts = torch.einsum("hn,nhd->hd", w, v.double()), torch.einsum("hn,nhd->hd", w, v.double().abs())
    err = (out[0].view(kvh, rep, 128).double() - want[:, None]).abs() / parts[:, None]
    assert float(err.max()) <= 2.0 ** -14.9, float(err.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,heads,kvh", [(8, 64, 8), (2, 64, 8)])
def test_nan_and_infinities_in_a_long_prompt(size, heads, kvh, dtype):
    """What is not finite in one prompt's values costs a look through them and not a sum a row: the other prompts' outputs keep
    their bits, no wait runs out, and the call stays within 10 ms (a row summed by itself takes some 2 ms, of 32 a warp)."""
    from deltazip_b200 import ops
    b = Batch([size] * 4, [16384, 9000, 16000, 5000], [20] * (4 * size), heads, kvh, dtype, seed=size)
    args = [b.qkv, b.k, b.v, i32(b.tables), i32(b.lens), i32(b.starts), i32(b.shared), size, 16384, heads, kvh, 16, SCALE]
    clean, rep = ops.shared_attention_decode(*args), heads // kvh
    for key, comp, value in ((3, 5, float("nan")), (7000, 9, float("inf")), (8999, 9, float("-inf")), (8000, 77, float("inf")),
                             (17, 100, float("-inf"))):
        for s in range(size, 2 * size):            # (page or copy: the same row for all, or one of each)
            b.v[b.slot(s, key), 3, comp] = value
    times = []
    for _ in range(3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        out = ops.shared_attention_decode(*args)
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    assert ops.read_status() == 0
    bad = torch.zeros_like(out, dtype=torch.bool).view(4 * size, kvh, rep, 128)
    bad[size:2 * size, 3, :, [5, 9, 77, 100]] = True
    assert torch.equal(out.view_as(bad)[~bad], clean.view_as(bad)[~bad])
    got = out.view_as(bad)[size:2 * size, 3]
    assert got[..., [5, 9]].isnan().all() and (got[..., 77] == float("inf")).all() and (got[..., 100] == float("-inf")).all()
    assert min(times) <= 10, times


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,heads,kvh", [(1, 1, 1), (8, 2, 2), (2, 8, 2), (9, 2, 2), (40, 2, 2)])
@pytest.mark.parametrize("below", [30, 45, 60, 100])
def test_infinities_far_below_the_maximum(below, size, heads, kvh, dtype):
    """A value of a key whose score is so far below the largest that its weight rounds to zero, in the part of that one and
    in another: what the definition gives does not depend on how many rows there are."""
    b = Batch([size, 1], [600, 40], [20] * (size + 1), heads, kvh, dtype, seed=below)
    b.qkv[:] = b.qkv[0].sign()
    b.k *= 0.02
    u = b.qkv[0, :128]
    b.qkv[:, :heads * 128] = u.repeat(heads)
    for s in range(size):
        b.k[b.slot(s, 100)] = (u.float() * (below / (128 * SCALE))).to(dtype)
        b.v[b.slot(s, 101), :, 7], b.v[b.slot(s, 599), :, 12], b.v[b.slot(s, 610), :, 20] = float("inf"), float("-inf"), float("inf")
        b.v[b.slot(s, 90), :, 33], b.v[b.slot(s, 580), :, 33], b.v[b.slot(s, 615), :, 50] = float("inf"), float("-inf"), float("nan")
    for longest in (600, 2000):
        out = b.run(longest=longest).view(size + 1, heads, 128)
        for s in range(size):
            want = b.want(s).view(heads, 128)
            assert want[:, [7, 12, 20]].isinf().all() and want[:, [33, 50]].isnan().all()
            odd = ~want.isfinite()
            assert int(odd.sum()) == 5 * heads and torch.equal(out[s].isfinite(), ~odd)
            assert torch.equal(torch.where(out[s].isnan(), 1., out[s].double())[odd], torch.where(want.isnan(), 1., want)[odd])
            err = (out[s].double()[~odd] - want[~odd]).norm() / want[~odd].norm()
            assert err <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rise", [0., 40.])
@pytest.mark.parametrize("groups,size,rep,kvh,block", [(37, 5, 8, 4, 16), (111, 5, 8, 4, 24), (222, 3, 8, 4, 24), (222, 2, 5, 8, 16), (222, 1, 3, 8, 9),
                                                       (222, 1, 1, 8, 16)])
def test_parts_of_several_rounds(groups, size, rep, kvh, block, rise, dtype):
    """Parts that are summed in several rounds, the last one short, in every form: tensor memory, teams of four and of two
    warps, a warp of sixteen and of eight rows, with and without whole tiles a page; the maximum the same or rising."""
    from deltazip_b200 import ops
    n, fresh, heads = 9001, 37, kvh * rep
    g = torch.Generator("cuda").manual_seed(groups + rep)
    pages = -(-(n + fresh) // block)
    u = torch.randn(128, generator=g, device="cuda").sign()
    q = torch.randn((size, heads, 128), generator=g, device="cuda") * 0.5 + u
    k = torch.randn((pages * block, kvh, 128), generator=g, device="cuda")
    k += (torch.linspace(0, rise, pages * block, device="cuda") / (128 * SCALE))[:, None, None] * u
    v = torch.randn((pages * block, kvh, 128), generator=g, device="cuda").to(dtype)
    q, k = q.to(dtype), k.to(dtype)
    qkv = torch.cat([q.reshape(size, -1), torch.zeros((size, 2 * kvh * 128), device="cuda", dtype=dtype)], 1).repeat(groups, 1)
    lens = [n + fresh * (s % 2) for s in range(size)]
    for shared in (n, 0):                          # with its group, and each by itself
        out = ops.shared_attention_decode(qkv, k, v, i32([list(range(pages))]).repeat(groups * size, 1), i32(lens * groups),
                                          i32(list(range(0, groups * size + 1, size))), i32([shared] * groups), size, shared, heads, kvh,
                                          block, SCALE).view(groups, size, heads, 128)
        assert torch.equal(out, out[:1].expand_as(out))
        for s, length in enumerate(lens):
            w = (torch.einsum("hrd,nhd->hrn", q[s].view(kvh, rep, 128).double(), k[:length].double()) * SCALE).softmax(-1)
            want = torch.einsum("hrn,nhd->hrd", w, v[:length].double()).reshape(heads, 128)
            err = (out[0, s].double() - want).norm() / want.norm()
            assert err <= TOL[dtype], (shared, s, float(err))


@pytest.mark.parametrize("size,heads,kvh,block", [(1, 8, 8, 16), (3, 32, 8, 16), (6, 32, 8, 16), (6, 32, 8, 40)])
def test_offsets_beyond_32_bits(size, heads, kvh, block):
    """A cache of 2^33 bytes and more, sequences in its last pages."""
    from deltazip_b200 import ops
    b = Batch([size, 2], [700, 100], [30] * (size + 2), heads, kvh, torch.float16, block=block, seed=block)
    have = b.k.shape[0] // block
    total = 2 ** 33 // (kvh * 256 * block) + have
    k, v = (torch.empty((total * block, kvh, 128), dtype=torch.float16, device="cuda") for _ in range(2))
    k[-have * block:], v[-have * block:] = b.k, b.v
    want = b.run()
    tables = [[p + total - have for p in row] for row in b.tables]
    got = ops.shared_attention_decode(b.qkv, k, v, i32(tables), i32(b.lens), i32(b.starts), i32(b.shared), size, 700, heads, kvh,
                                      block, SCALE)
    assert torch.equal(got, want)
