"""Beam search's selection against log-softmax and a sort in 64 bits: vocabularies around a thread's, a warp's and a
piece's elements, odd strides and addresses, ragged and empty groups, masks, infinities, NaN and equal logits.

Tolerance of a score: log sum exp is off by at most 55 half steps of 32 bits -- two units of the exponential (4), the
rounding of a difference of up to 20 (20), 31 additions within a thread (31); everything behind is 64-bit -- and the score
by half a step of its own: 55 * 2^-24 + |score| * 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def reference(logits, scores, starts, k):
    """Per group [(score, row, token)] best first, every place filled, in 64 bits."""
    out = []
    for a, b in zip(starts, starts[1:]):
        z = logits[a:b].double()
        z = torch.where(z.isnan(), -INF, z)
        value = scores[a:b, None].double() + torch.log_softmax(z, 1)
        dead = (z.max(1).values == -INF if b > a and z.shape[1] else torch.zeros(b - a, dtype=torch.bool, device="cuda")) \
            | ~scores[a:b].isfinite()
        value = torch.where(dead[:, None], -INF, value).reshape(-1)
        order = torch.sort(value, descending=True, stable=True)[1][:k]
        got = [(float(value[i]), a + int(i) // z.shape[1], int(i) % z.shape[1]) for i in order]
        out.append(got + [(-INF, -1, -1)] * (k - len(got)))
    return out


def check(got, want):
    for g, group in enumerate(want):
        assert got.rows[g].tolist() == [r for _, r, _ in group], g
        assert got.tokens[g].tolist() == [t for _, _, t in group], g
        for s, (w, _, _) in zip(got.scores[g].tolist(), group):
            assert s == w or abs(s - w) <= 55 * 2.0 ** -24 + abs(w) * 2.0 ** -24, (s, w)


def inputs(rows, vocab, dtype, seed, std=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g, device="cuda") * std).to(dtype), -10 * torch.rand(rows, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 255, 256, 257, 2047, 2048, 2049, 8191, 8200, 32000, 50001])
@pytest.mark.parametrize("k", [1, 8, 33, 128])
def test_vocabularies(vocab, k, dtype):
    from deltazip_b200 import ops
    starts = [0, 3, 4, 4, 9]
    logits, scores = inputs(9, vocab, dtype, vocab + k)
    check(ops.beam_select(logits, scores, i32(starts), k), reference(logits, scores, starts, k))


@pytest.mark.parametrize("rows,vocab,k", [(1, 700, 4), (200, 9000, 16), (600, 300, 20), (37, 131072, 64)])
def test_rows(rows, vocab, k):
    """Few rows in small pieces, many in large ones, a group of more rows than the second launch has threads."""
    from deltazip_b200 import ops
    logits, scores = inputs(rows, vocab, torch.float32, rows)
    for starts in ([0, rows], [0, rows // 3, rows]):
        check(ops.beam_select(logits, scores, i32(starts), k), reference(logits, scores, starts, k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 3), (8, 8)])
def test_strides_and_addresses(pad, shift, dtype):
    from deltazip_b200 import ops
    wide, scores = inputs(7, 5000 + pad + shift, dtype, pad)
    logits = wide[:, shift:shift + 5000]
    check(ops.beam_select(logits, scores, i32([0, 2, 7]), 12), reference(logits, scores, [0, 2, 7], 12))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 5000, 20000])
def test_equal_logits(vocab, dtype):
    """All alike; alike but for a few; few values: the lower token and, at equal scores, the lower row come first."""
    from deltazip_b200 import ops
    logits = torch.zeros((6, vocab), dtype=dtype, device="cuda")
    scores = torch.full((6,), -1.5, device="cuda")
    logits[2, 17] = logits[3, 17] = logits[3, 30] = 2
    logits[4:] = torch.randint(0, 3, (2, vocab), generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(dtype)
    logits[5] = logits[4]
    starts = [0, 2, 4, 6]
    check(ops.beam_select(logits, scores, i32(starts), 24), reference(logits, scores, starts, 24))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("left", [0, 1, 5, 300])
def test_masks(left, dtype):
    """All but a few tokens masked, by -inf, by the type's lowest value, by NaN; rows of which nothing is left."""
    from deltazip_b200 import ops
    vocab, k = 21000, 16
    logits, scores = inputs(6, vocab, dtype, left)
    keep = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    keep[9000:9000 + left] = True
    for row, mask in enumerate((-INF, torch.finfo(dtype).min, float("nan"), -INF)):
        logits[row, ~keep] = mask
    starts = [0, 1, 2, 4, 6]
    check(ops.beam_select(logits, scores, i32(starts), k), reference(logits, scores, starts, k))


def test_rows_that_are_not_continued():
    from deltazip_b200 import ops
    logits, scores = inputs(8, 900, torch.float32, 3)
    scores[0], scores[3], scores[4], scores[6:] = -INF, float("nan"), INF, -INF
    starts = [0, 3, 6, 8]
    check(ops.beam_select(logits, scores, i32(starts), 10), reference(logits, scores, starts, 10))


def test_infinite_logits_share_the_probability():
    from deltazip_b200 import ops
    logits, scores = inputs(2, 30000, torch.float32, 4)
    logits[0, [5, 29000]] = INF
    logits[1, 77] = INF
    got = ops.beam_select(logits, scores, i32([0, 2]), 3)
    want = sorted([(float(scores[0]) - 0.6931471805599453, 0, 5), (float(scores[0]) - 0.6931471805599453, 0, 29000),
                   (float(scores[1]), 1, 77)], key=lambda c: (-c[0], c[1], c[2]))
    check(got, [want])


def test_ordered_vocabularies():
    """Logits that fall or rise with the token, and peaks inside one thread's elements: every candidate in one place."""
    from deltazip_b200 import ops
    vocab = 16384
    logits = torch.stack([torch.arange(vocab, device="cuda") * s for s in (-0.01, 0.01)]).float()
    logits = torch.cat([logits, torch.zeros((1, vocab), device="cuda")])
    logits[2, :8] = logits[2, 1024:1032] = 9
    starts, scores = [0, 1, 2, 3], torch.zeros(3, device="cuda")
    check(ops.beam_select(logits, scores, i32(starts), 100), reference(logits, scores, starts, 100))


def test_empty():
    from deltazip_b200 import ops
    got = ops.beam_select(torch.empty((0, 50), device="cuda"), torch.empty(0, device="cuda"), i32([0, 0, 0]), 4)
    assert got.tokens.tolist() == [[-1] * 4] * 2 and got.rows.tolist() == [[-1] * 4] * 2 and bool((got.scores == -INF).all())
    got = ops.beam_select(torch.empty((0, 50), device="cuda"), torch.empty(0, device="cuda"), i32([0]), 4)
    assert got.tokens.shape == (0, 4)


def test_same_bits_again_and_in_a_graph():
    """On a side stream, captured twice, the graphs replayed in turn with other inputs: bit for bit what a call gives."""
    from deltazip_b200 import ops
    side = torch.cuda.Stream()
    cases = [(inputs(5, 33000, torch.float16, s), i32([0, 2, 5])) for s in (1, 2)]
    want = [ops.beam_select(x, c, st, 9) for (x, c), st in cases]
    bufs = [[t.clone() for t in cases[0][0]], [t.clone() for t in cases[0][0]]]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(ops.beam_select(*b, cases[0][1], 9))
        graphs.append(g)
    for t, n in zip(bufs[1], cases[1][0]):
        t.copy_(n)
    for rep in range(3):
        graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_refusals():
    from deltazip_b200 import ops
    from deltazip_b200._lib import DeltaZipError
    logits, scores, starts = torch.zeros((4, 10), device="cuda"), torch.zeros(4, device="cuda"), i32([0, 4])
    for bad in (dict(k=0), dict(k=129), dict(k=-1)):
        with pytest.raises((DeltaZipError, RuntimeError)):
            ops.beam_select(logits, scores, starts, bad["k"])
    for args in ((logits.t(), torch.zeros(10, device="cuda"), starts), (logits, scores[:3], starts), (logits, scores.half(), starts),
                 (logits, scores, starts.long()), (logits.double(), scores, starts), (logits[0], scores, starts),
                 (logits, scores, starts[:0]), (logits.int(), scores, starts)):
        with pytest.raises(ValueError):
            ops.beam_select(*args, 4)
    with pytest.raises(DeltaZipError):
        ops.beam_select(logits[:, :0], scores, starts, 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab,k", [(2, 2), (40, 8), (5000, 24), (20000, 100)])
def test_zeros_of_both_signs_are_equal(vocab, k, dtype):
    """Logits multiplied by a mask: zeros of both signs among the best, at the k-th place and in all places; the lower token
    comes first whatever its sign."""
    from deltazip_b200 import ops
    g = torch.Generator("cuda").manual_seed(vocab)
    signs = torch.where(torch.rand((6, vocab), generator=g, device="cuda") < 0.5, -1., 1.)
    logits = (torch.zeros((6, vocab), device="cuda") * signs).to(dtype)
    logits[0, :vocab // 2], logits[0, vocab // 2:] = -0., 0.
    logits[3:] = torch.where(torch.rand((3, vocab), generator=g, device="cuda") < 0.7, logits[3:].float(), -signs[3:].abs() * 2).to(dtype)
    logits[4, vocab // 3] = 1
    assert bool((logits.signbit() & (logits == 0)).any())
    scores = torch.tensor([-1.5, -1.5, -0., 0., -1., -1.], device="cuda")
    for starts in ([0, 1, 3, 6], [0, 6]):
        check(ops.beam_select(logits, scores, i32(starts), k), reference(logits, scores, starts, k))
    logits[:] = -1                                 # one token of a row has the whole probability: scores of both signs of zero
    logits[:, 1] = INF
    got = ops.beam_select(logits, torch.tensor([-0., 0., -0., 0., -0., 0.], device="cuda"), i32([0, 6]), 6)
    assert got.rows.tolist() == [list(range(6))] and got.tokens.tolist() == [[1] * 6] and not got.scores.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [-3000., 1000., 50000.])
def test_nan_among_large_logits(offset, dtype):
    """A NaN among the logits of some threads, of all, and of all but the first: the others' sum is as exact as without it."""
    from deltazip_b200 import ops
    vocab = 20000
    logits, scores = inputs(6, vocab, torch.float32, 7)
    logits = (logits + offset).to(dtype)
    every = torch.arange(vocab, device="cuda")
    for row, nan in enumerate((every % 997 == 3, every % 3 == 1, every > 0, every % 8 == 7, every < vocab - 40)):
        logits[row, nan] = float("nan")
    starts = [0, 1, 2, 3, 4, 5, 6]
    check(ops.beam_select(logits, scores, i32(starts), 12), reference(logits, scores, starts, 12))


@pytest.mark.parametrize("rows,vocab,dtype", [(3, 2 ** 30, torch.bfloat16), (9, 2 ** 28 + 3, torch.float32)])
def test_offsets_beyond_32_bits(rows, vocab, dtype):
    """The largest vocabulary, and rows that begin behind 2^32 bytes."""
    from deltazip_b200 import ops
    g = torch.Generator("cuda").manual_seed(rows)
    logits = torch.empty((rows, vocab), dtype=dtype, device="cuda")
    for row in logits:
        row.normal_(0, 1, generator=g)
    for row in range(rows):                        # the best in places of their own
        logits[row, [vocab - 1 - row, 7, vocab // 2 + row]] = torch.tensor([30. - row, 29.5 - row, 31. - row], device="cuda").to(dtype)
    scores = -torch.arange(rows, device="cuda").float()
    got = ops.beam_select(logits, scores, i32([0, rows - 1, rows]), 6)
    for group, (a, b) in enumerate(((0, rows - 1), (rows - 1, rows))):
        want = []
        for row in range(a, b):
            z, lse = logits[row], 0.
            for part in z.split(2 ** 27):
                lse += float(part.double().exp().sum())
            top = z.topk(8)
            lse = float(torch.log(torch.tensor(lse, dtype=torch.float64)))
            want += [(float(scores[row]) + float(x) - lse, row, int(t)) for x, t in zip(*top)]
        want.sort(key=lambda c: (-c[0], c[1], c[2]))
        assert got.rows[group, :3].tolist() == [r for _, r, _ in want[:3]]
        assert got.tokens[group, :3].tolist() == [t for _, _, t in want[:3]]
        for s, (w, _, _) in zip(got.scores[group, :3].tolist(), want):
            assert abs(s - w) <= 55 * 2.0 ** -24 + abs(w) * 2.0 ** -24
