"""Copies between pages of all pools, bit for bit against indexing: row sizes that make every unit from 16 bytes to one,
few and many pairs, partly filled pages, chains, cycles, doubled destinations and pairs that are left out."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def random_pools(shapes, pages, rows, seed=0):
    """shapes: (size of a row..., type); values from random bits of small integers, exact in every type."""
    g = torch.Generator("cuda").manual_seed(seed)
    return [torch.randint(0, 200, (pages * rows, *s[:-1]), generator=g, device="cuda").to(s[-1]) for s in shapes]


def expected(pools, per, src, dst, rows=None):
    n = pools[0].shape[0] // per
    out = []
    for p in pools:
        old = p.view(n, per, *p.shape[1:])
        new = old.clone()
        for i, (s, d) in enumerate(zip(src, dst)):
            if 0 <= s < n and 0 <= d < n:
                new[d] = old[d]                    # the last pair counts, not what an earlier one left
                m = per if rows is None else max(0, min(per, rows[i]))
                new[d, :m] = old[s, :m]
        out.append(new.view(p.shape))
    return out


def run(pools, per, src, dst, rows=None):
    from deltazip_b200 import ops
    want = expected(pools, per, src, dst, rows)
    handle = ops.PagePools(pools, per)
    ops.copy_pages(handle, i32(src), i32(dst), None if rows is None else i32(rows))
    for got, w in zip(pools, want):
        assert torch.equal(got, w)


SHAPES = [
    [(8, 128, torch.float16), (8, 128, torch.float16)],
    [(1, 576, torch.bfloat16)],
    [(3, 4, torch.float16), (5, torch.float32), (7, torch.int8), (6, torch.int16), (2, 64, torch.float32)],
    [(1, torch.float32), (33, 40, 24, torch.float32)],
]


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("per", [1, 5, 16])
@pytest.mark.parametrize("pairs", [1, 2, 9, 30])
def test_apart(shapes, per, pairs):
    import random
    rng = random.Random(per + pairs)
    pages = list(range(64))
    rng.shuffle(pages)
    dst, rest = pages[:pairs], pages[pairs:]
    src = [rng.choice(rest) for _ in dst]
    run(random_pools(shapes, 64, per), per, src, dst)
    run(random_pools(shapes, 64, per), per, src, dst, [rng.randint(-1, per + 1) for _ in dst])


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("per", [1, 16])
@pytest.mark.parametrize("pairs", [2, 7, 40, 300])
def test_at_once(shapes, per, pairs):
    """Any pages on both sides: what is read is what was there before the call."""
    import random
    rng = random.Random(per + pairs)
    src, dst = [rng.randrange(320) for _ in range(pairs)], rng.sample(range(320), pairs)
    run(random_pools(shapes, 320, per), per, src, dst)
    run(random_pools(shapes, 320, per), per, src, dst, [rng.randint(0, per) for _ in dst])


def test_cycles_and_chains():
    pools = lambda: random_pools(SHAPES[0], 16, 4)
    run(pools(), 4, [0, 1, 2, 3], [1, 2, 3, 0])
    run(pools(), 4, [3, 4, 5], [4, 5, 6])
    run(pools(), 4, [5, 4, 3], [6, 5, 4])
    run(pools(), 4, [7, 7, 2], [7, 3, 7])
    run(pools(), 4, list(range(16)), list(range(15, -1, -1)))


@pytest.mark.parametrize("pairs", [3, 50])
def test_pairs_left_out_and_doubled(pairs):
    import random
    rng = random.Random(pairs)
    src = [rng.randrange(-3, 24) for _ in range(pairs)]
    dst = [rng.randrange(-3, 24) for _ in range(pairs)]
    run(random_pools(SHAPES[2], 20, 3), 3, src, dst)
    run(random_pools(SHAPES[2], 20, 3), 3, src, dst, [rng.randint(0, 3) for _ in dst])
    run(random_pools(SHAPES[0], 20, 3), 3, [1, 2, 3], [9, 9, 9], [3, 1, 2])


def test_many_pairs():
    """As many as a call takes, apart and as one permutation."""
    import random

    from deltazip_b200 import ops
    n = ops.copy_pages_max_pairs()
    rng = random.Random(1)
    order = rng.sample(range(n), n)
    run(random_pools([(24, torch.float32)], n, 1), 1, order, list(range(n)))
    run(random_pools([(2, 64, torch.float16)], 2 * n, 2), 2, list(range(n)), [n + i for i in order])


def test_large_pools_pass_32_bits():
    """Pages beyond 4 GB of a pool, in both forms."""
    pages, per = 2200, 16
    pool = torch.zeros((pages * per, 32, 128, 16), dtype=torch.float16, device="cuda")
    pool[(pages - 1) * per:] = 3
    pool[(pages - 2) * per:(pages - 1) * per] = 5
    from deltazip_b200 import ops
    handle = ops.PagePools([pool], per)
    ops.copy_pages(handle, i32([pages - 1]), i32([0]))
    ops.copy_pages(handle, i32([pages - 1, pages - 2]), i32([pages - 2, pages - 1]))
    for page, want in ((0, 3), (pages - 1, 5), (pages - 2, 3), (1, 0)):
        assert bool((pool[page * per:(page + 1) * per] == want).all())


def test_views_that_start_anywhere():
    """Pools that start at odd addresses of a buffer."""
    from deltazip_b200 import ops
    flat = torch.randint(0, 100, (4000,), device="cuda").to(torch.int16)
    for shift in (1, 2, 4, 8):
        pool = flat[shift:shift + 40 * 16].view(40, 16)
        want, rest = expected([pool], 4, [0, 3, 9], [9, 1, 0])[0], flat.clone()
        ops.copy_pages(ops.PagePools([pool], 4), i32([0, 3, 9]), i32([9, 1, 0]))
        assert torch.equal(pool, want) and torch.equal(flat[:shift], rest[:shift]) and torch.equal(flat[shift + 640:], rest[shift + 640:])


def test_nothing_to_do():
    from deltazip_b200 import ops
    pool = random_pools(SHAPES[0], 8, 2)[0]
    was = pool.clone()
    ops.copy_pages(ops.PagePools([pool], 2), i32([]), i32([]))
    ops.copy_pages(ops.PagePools([], 2), i32([1]), i32([2]))
    ops.copy_pages(ops.PagePools([torch.empty((16, 3, 0), device="cuda")], 2), i32([1]), i32([2]))
    ops.copy_pages(ops.PagePools([pool, torch.empty((16, 3, 0), device="cuda")], 2), i32([1]), i32([1]))
    assert torch.equal(pool, was)


def test_captured():
    """The indices of a replayed graph are read when it runs; two graphs share the pools."""
    from deltazip_b200 import ops
    pools = random_pools(SHAPES[3], 12, 1)
    handle = ops.PagePools(pools, 1)
    src, dst = i32([0, 1, 2]), i32([4, 5, 6])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.copy_pages(handle, src, dst)
        graphs.append(g)
    want = expected(expected(pools, 1, [0, 1, 2], [4, 5, 6]), 1, [4, 5, 5], [5, 4, 8])
    graphs[0].replay()
    src.copy_(i32([4, 5, 5]))
    dst.copy_(i32([5, 4, 8]))
    graphs[1].replay()
    for got, w in zip(pools, want):
        assert torch.equal(got, w)


def test_refusals():
    from deltazip_b200 import ops
    from deltazip_b200._lib import DeltaZipError
    pool = torch.zeros((16, 8), device="cuda")
    handle = ops.PagePools([pool], 4)
    for bad in ((i32([1]), i32([1, 2]), None), (i32([1]).long(), i32([1]), None), (i32([1, 2]), i32([3, 0]), i32([1])),
                (i32([1, 2, 3, 0])[::2], i32([1, 2]), None), (i32([[1]]), i32([[1]]), None)):
        with pytest.raises(ValueError):
            ops.copy_pages(handle, *bad)
    n = ops.copy_pages_max_pairs() + 1
    with pytest.raises(DeltaZipError):
        ops.copy_pages(handle, i32([0] * n), i32([1] * n))
    for tensors, per in (([pool], 3), ([pool], 0), ([pool.t()], 4), ([pool, pool[:8]], 4), ([pool.cpu()], 4),
                         ([torch.zeros((), device="cuda")], 1), ([pool, pool], 4), ([pool[:8], pool[4:12]], 4)):
        with pytest.raises(ValueError):
            ops.PagePools(tensors, per)


def test_offsets_beyond_32_bits():
    """Pages behind 2^33 bytes of a pool, in the form that reads all pairs first and in the one that does not."""
    from deltazip_b200 import ops
    pages, size = 140000, 64 * 1024
    pool = torch.empty((pages, size), dtype=torch.uint8, device="cuda")
    last = [pages - 1 - i for i in range(6)]
    for i, p in enumerate(last):
        pool[p] = i + 1
    handle = ops.PagePools([pool], 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    ops.copy_pages(handle, ints(last[:2] + [5]), ints(last[2:4] + [6]))
    assert [int(pool[p].float().mean()) for p in last] == [1, 2, 1, 2, 5, 6]
    ops.copy_pages(handle, ints([last[0], last[5]]), ints([last[5], last[0]]))
    assert [int(pool[p].float().mean()) for p in last] == [6, 2, 1, 2, 5, 1]
    assert all(bool((pool[p] == pool[p, 0]).all()) for p in last)
