"""Beam search over paged caches, as cases whose time can be taken: the selection over beams and vocabulary, the copying
of cache pages and recurrent states, and decode attention of sequences that share their first pages.

A case is a dict of plain values with a "kind".  `run` computes it in plain torch, or through the package's operators
where `own` is true; `exact` says what the definition gives in 64 bits."""
from __future__ import annotations

import random

import torch

own = False                             # whether run() calls the package's operators

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
HEAD = 128                              # head size of the paged decode kernels
BLOCK = 16                              # tokens of a cache page
I32 = torch.int32


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + 12345)


def _normal(gen, *shape, dtype=torch.float32, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0, std, generator=gen)


def _rng(c: dict) -> random.Random:
    """Lengths, groups and pages belong to the case, so that its work is the same whatever the seed."""
    return random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=I32).to(DEV)


def _groups(c: dict, rng: random.Random) -> list:
    """Sequences of every prompt: its beams, or, where beams have ended or prompts differ, between one and that many."""
    if not c["ragged"]:
        return [c["beams"]] * c["prompts"]
    sizes = [rng.randint(1, c["beams"]) for _ in range(c["prompts"])]
    sizes[rng.randrange(c["prompts"])] = c["beams"]
    return sizes


def _starts(sizes: list) -> list:
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------------------------
# kind "select": the best continuations of every prompt's beams
# ---------------------------------------------------------------------------

def _prepare_select(c: dict, seed: int) -> dict:
    rng, gen = _rng(c), _gen(seed)
    starts = _starts(_groups(c, rng))
    rows = starts[-1]
    logits = _normal(gen, rows, c["vocab"], std=2.5)
    if c["masked"]:                     # constrained decoding: what the grammar forbids has the lowest logit there is
        banned = torch.rand((rows, c["vocab"]), generator=gen, device=DEV) < 0.9
        logits = logits.masked_fill_(banned, float("-inf"))
        logits[1::3] = logits[1::3].clamp_(min=torch.finfo(TYPES[c["dtype"]]).min)
    scores = -20 * torch.rand(rows, generator=gen, device=DEV)
    return {"c": c, "logits": logits.to(TYPES[c["dtype"]]), "scores": scores, "starts": _ints(starts)}


def _run_select(s: dict) -> dict:
    c, k = s["c"], s["c"]["keep"]
    if own:
        from deltazip_b200 import ops
        got = ops.beam_select(s["logits"], s["scores"], s["starts"], k)
        return {"scores": got.scores, "rows": got.rows, "tokens": got.tokens}
    logits = s["logits"].float()
    logits = torch.where(logits.isnan(), float("-inf"), logits)
    best, tokens = logits.sort(dim=1, descending=True, stable=True)
    best, tokens = best[:, :k].double(), tokens[:, :k]
    top = best[:, :1]                                                       # borders between beams are held in 64 bits
    lse = top + torch.log(torch.exp(logits.double() - top).sum(1, keepdim=True))
    value = s["scores"].double()[:, None] + (best - lse)
    rows = s["starts"][:-1, None].long() + torch.arange(c["beams"], device=DEV)
    live = rows < s["starts"][1:, None]
    rows = rows.clamp(max=logits.shape[0] - 1)
    flat = torch.where(live[:, :, None], value[rows], float("-inf")).flatten(1)
    order = flat.sort(dim=1, descending=True, stable=True)[1][:, :k]
    return {"scores": flat.gather(1, order).float(), "rows": rows.gather(1, order // best.shape[1]).to(I32),
            "tokens": tokens[rows].flatten(1).gather(1, order).to(I32)}


def _exact_select(s: dict) -> dict:
    k, out = s["c"]["keep"], {"scores": [], "rows": [], "tokens": []}
    starts = s["starts"].tolist()
    for a, b in zip(starts, starts[1:]):
        z = s["logits"][a:b].double().nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
        joint = (s["scores"][a:b, None].double() + z - torch.logsumexp(z, 1, keepdim=True)).reshape(-1)
        at = torch.argsort(joint, descending=True, stable=True)[:k]
        out["scores"].append(joint[at])
        out["rows"].append(a + at // z.shape[1])
        out["tokens"].append(at % z.shape[1])
    return {name: torch.stack(v) for name, v in out.items()}


def _work_select(c: dict) -> dict:
    rows = sum(_groups(c, _rng(c)))
    n = rows * c["vocab"]
    return {"bytes": n * BYTES[c["dtype"]] + 4 * rows + 12 * c["prompts"] * c["keep"], "flops": 4 * n}


# ---------------------------------------------------------------------------
# kind "pages": copies between pages of all pools of a cache, and "states": a new order of recurrent states
# ---------------------------------------------------------------------------

def _pairs(c: dict):
    """(source pages, destination pages, rows of each that are in use)."""
    rng = _rng(c)
    if c["kind"] == "states":           # every sequence goes on from the state of one of its prompt's beams
        src = [g + rng.randrange(c["beams"]) for g in range(0, c["slots"], c["beams"]) for _ in range(c["beams"])]
        return src, list(range(c["slots"])), None
    pages = list(range(c["pages"]))
    rng.shuffle(pages)
    dst, parents = pages[:c["copies"]], pages[c["copies"]:]
    if c["compact"]:                    # whole pages from anywhere to free ones
        return parents[:c["copies"]], dst, None
    src = [rng.choice(parents[:max(1, c["copies"] // 2)]) for _ in dst]     # a page that is written on by several beams
    return src, dst, [rng.randint(1, BLOCK) for _ in dst]


def _prepare_copy(c: dict, seed: int) -> dict:
    gen = _gen(seed)
    if c["kind"] == "states":
        shapes = [(c["slots"], c["heads"], c["dim"], c["vdim"])] * c["runs"]
        if c["normalised"]:
            shapes += [(c["slots"], c["heads"], c["dim"])] * c["runs"] + [(c["slots"], c["heads"])] * c["runs"]
    else:
        shapes = [(c["pages"] * BLOCK, c["kv_heads"], c["head"])] * (2 * c["layers"])
    pools = [_normal(gen, *shape, dtype=TYPES[c["dtype"]]) for shape in shapes]
    src, dst, rows = _pairs(c)
    per = 1 if c["kind"] == "states" else BLOCK
    s = {"c": c, "pools": pools, "per": per, "src": _ints(src), "dst": _ints(dst), "rows": None if rows is None else _ints(rows)}
    if own:                             # the handle that a cache keeps for its pools
        from deltazip_b200 import ops
        s["handle"] = ops.PagePools(pools, per)
    return s


def _run_copy(s: dict) -> list:
    if own:
        from deltazip_b200 import ops
        ops.copy_pages(s["handle"], s["src"], s["dst"], s["rows"])
        return s["pools"]
    inner = torch.arange(s["per"], device=DEV)
    src, dst = (t.long()[:, None] * s["per"] + inner for t in (s["src"], s["dst"]))
    if s["rows"] is not None:           # rows that are not in use stay as they are
        src = torch.where(inner < s["rows"][:, None], src, dst)
    for pool in s["pools"]:
        pool[dst.flatten()] = pool[src.flatten()]
    return s["pools"]


def _exact_copy(s: dict) -> list:
    c, per = s["c"], s["per"]
    src, dst, rows = _pairs(c)
    out = []
    for pool in s["pools"]:
        old = pool.view(-1, per, *pool.shape[1:])
        new = old.clone()
        for i, (a, b) in enumerate(zip(src, dst)):
            n = per if rows is None else rows[i]
            new[b, :n] = old[a, :n]
        out.append(new.view(pool.shape))
    return out


def _work_copy(c: dict) -> dict:
    src, _, rows = _pairs(c)
    if c["kind"] == "states":
        sizes = c["dim"] * c["vdim"] + (c["dim"] + 1 if c["normalised"] else 0)
        one, units = c["runs"] * c["heads"] * sizes, len(src)
    else:
        one, units = 2 * c["layers"] * c["kv_heads"] * c["head"], BLOCK * len(src) if rows is None else sum(rows)
    return {"bytes": 2 * one * units * BYTES[c["dtype"]] + 8 * len(src), "flops": 0}


# ---------------------------------------------------------------------------
# kind "attention": one new token of every beam against its prompt's pages and its own
# ---------------------------------------------------------------------------

def _lengths(c: dict):
    """(sequences of every prompt, its shared length, own length of every sequence)."""
    rng = _rng(c)
    sizes = _groups(c, rng)
    shared = [rng.randint(max(1, c["shared"] // (4 * BLOCK)), c["shared"] // BLOCK) * BLOCK for _ in sizes]
    shared[rng.randrange(len(sizes))] = c["shared"]
    fresh = [rng.randint(max(1, c["own"] // 2), c["own"]) for _ in sizes]   # beams of a prompt are equally long
    return sizes, shared, [n for size, n in zip(sizes, fresh) for _ in range(size)]


def _prepare_attention(c: dict, seed: int) -> dict:
    rng, gen, dt = random.Random(seed * 31 + 5), _gen(seed), TYPES[c["dtype"]]
    sizes, shared, fresh = _lengths(c)
    group = [g for g, size in enumerate(sizes) for _ in range(size)]
    need = [n // BLOCK for n in shared] + [-(-n // BLOCK) for n in fresh]
    pool, tables = list(range(sum(need))), []
    rng.shuffle(pool)
    cut = _starts(need)
    wide = max(need[g] + need[len(sizes) + i] for i, g in enumerate(group))
    for i, g in enumerate(group):
        at = len(sizes) + i
        pages = pool[cut[g]:cut[g + 1]] + pool[cut[at]:cut[at + 1]]
        tables.append(pages + [0] * (wide - len(pages)))
    heads, kvh, n = c["heads"], c["kv_heads"], len(group)
    rnd = lambda *shape: _normal(gen, *shape, dtype=dt)
    return {"c": c, "qkv": rnd(n, (heads + 2 * kvh) * HEAD), "k": rnd(sum(need) * BLOCK, kvh, HEAD),
            "v": rnd(sum(need) * BLOCK, kvh, HEAD), "tables": _ints(tables), "starts": _ints(_starts(sizes)),
            "shared": _ints(shared), "lens": _ints([shared[g] + f for g, f in zip(group, fresh)]), "scale": HEAD ** -0.5,
            "most": max(sizes), "longest": max(shared), "group": _ints(group)}


def _run_attention(s: dict) -> torch.Tensor:
    c = s["c"]
    heads, kvh = c["heads"], c["kv_heads"]
    if own:
        from deltazip_b200 import ops
        return ops.shared_attention_decode(s["qkv"], s["k"], s["v"], s["tables"], s["lens"], s["starts"], s["shared"], s["most"],
                                           s["longest"], heads, kvh, BLOCK, s["scale"])
    n, wide = s["tables"].shape
    t = torch.arange(wide * BLOCK, device=DEV)
    page = s["tables"].long().repeat_interleave(BLOCK, 1)
    first = page[s["starts"][:-1].long()][s["group"].long()]
    at = torch.where(t < s["shared"].long()[s["group"].long()][:, None], first, page) * BLOCK + t % BLOCK
    q = s["qkv"][:, :heads * HEAD].float().view(n, kvh, heads // kvh, HEAD) * s["scale"]
    x = torch.matmul(q, s["k"][at].float().permute(0, 2, 3, 1))             # [sequence, key head, query head, key]
    x = x.masked_fill(t >= s["lens"].long()[:, None, None, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p, s["v"][at].float().permute(0, 2, 1, 3)) / p.sum(-1, keepdim=True)
    return o.reshape(n, heads * HEAD).to(s["qkv"].dtype)


def _exact_attention(s: dict) -> torch.Tensor:
    c = s["c"]
    heads, kvh = c["heads"], c["kv_heads"]
    rep, out = heads // kvh, []
    tables, lens, starts, group = (s[k].cpu() for k in ("tables", "lens", "starts", "group"))
    for i in range(len(lens)):
        n, g = int(lens[i]), int(group[i])
        prefix = int(s["shared"][g])
        pos = torch.arange(n)
        pages = torch.where(pos < prefix, tables[int(starts[g])].long()[pos // BLOCK], tables[i].long()[pos // BLOCK])
        at = (pages * BLOCK + pos % BLOCK).to(DEV)
        k, v = s["k"][at].double(), s["v"][at].double()
        q = s["qkv"][i, :heads * HEAD].double().view(kvh, rep, HEAD)
        p = torch.softmax(torch.einsum("hrd,nhd->hrn", q, k) * s["scale"], -1)
        out.append(torch.einsum("hrn,nhd->hrd", p, v).reshape(-1))
    return torch.stack(out)


def _work_attention(c: dict) -> dict:
    sizes, shared, fresh = _lengths(c)
    row = 2 * c["kv_heads"] * HEAD * BYTES[c["dtype"]]
    keys = sum(shared[g] for g, size in enumerate(sizes) for _ in range(size)) + sum(fresh)
    return {"bytes": (sum(shared) + sum(fresh)) * row + 2 * len(fresh) * c["heads"] * HEAD * BYTES[c["dtype"]],
            "flops": 4 * c["heads"] * HEAD * keys}


# ---------------------------------------------------------------------------

_KINDS = {"select": (_prepare_select, _run_select, _exact_select, _work_select),
          "pages": (_prepare_copy, _run_copy, _exact_copy, _work_copy),
          "states": (_prepare_copy, _run_copy, _exact_copy, _work_copy),
          "attention": (_prepare_attention, _run_attention, _exact_attention, _work_attention)}


def _select(prompts, beams, vocab, keep, dtype="fp32", ragged=False, masked=False, **name) -> dict:
    return dict(name, kind="select", prompts=prompts, beams=beams, vocab=vocab, keep=keep, dtype=dtype, ragged=ragged, masked=masked)


def _pages(layers, kv_heads, pages, copies, head=HEAD, dtype="fp16", compact=False, **name) -> dict:
    return dict(name, kind="pages", layers=layers, kv_heads=kv_heads, head=head, pages=pages, copies=copies, dtype=dtype,
                compact=compact)


def _states(runs, heads, dim, vdim, slots, beams, normalised, **name) -> dict:
    return dict(name, kind="states", runs=runs, heads=heads, dim=dim, vdim=vdim, slots=slots, beams=beams, normalised=normalised,
                dtype="fp32")


def _attention(prompts, beams, heads, kv_heads, shared, own_keys, dtype="fp16", ragged=False, **name) -> dict:
    return dict(name, kind="attention", prompts=prompts, beams=beams, heads=heads, kv_heads=kv_heads, shared=shared, own=own_keys,
                dtype=dtype, ragged=ragged)


def listed() -> list:
    return [
        # one request with four beams: latency is all there is
        _select(1, 4, 32000, 8, name="select_one_prompt"),
        # a serving batch of eight beams a prompt over the vocabulary of the decoders here
        _select(16, 8, 32000, 16, name="select_batch"),
        # a large vocabulary in 16 bits, groups in which some beams have ended, wide beams
        _select(32, 16, 131072, 32, dtype="bf16", ragged=True, name="select_wide"),
        # constrained decoding over a vocabulary of odd size: most tokens forbidden
        _select(12, 5, 50001, 10, dtype="fp16", ragged=True, masked=True, name="select_masked_odd"),
        # a beam that forks inside a page of a small model
        _pages(2, 8, 64, 1, name="pages_one"),
        # the forks of one step of a serving batch: partly filled pages of eight layers of a 7B decoder
        _pages(8, 32, 512, 96, name="pages_forks"),
        # a cache with few key heads whose live pages move together
        _pages(8, 8, 4096, 1500, dtype="bf16", compact=True, name="pages_compact"),
        # matrix memories of a recurrent decoder follow the beams that were chosen
        _states(4, 16, 128, 128, 64, 8, True, name="states_reorder"),
        # one prompt with four beams, 32 heads
        _attention(1, 4, 32, 32, 512, 64, name="attention_one_prompt"),
        # eight beams on each of sixteen prompts, 32 heads as in a 7B decoder
        _attention(16, 8, 32, 32, 2048, 128, name="attention_batch"),
        # long prompts with grouped query heads: 64 on 8
        _attention(4, 8, 64, 8, 16384, 200, dtype="bf16", name="attention_grouped_long"),
        # prompts with between one and twelve beams that have gone on for long, 40 heads as in a 13B decoder
        _attention(12, 12, 40, 40, 1008, 700, dtype="bf16", ragged=True, name="attention_uneven"),
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    """Spread over the logarithm of the range."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["select", "pages", "states", "attention"])
    if kind == "select":
        beams, vocab = rng.randint(1, 16), _log(rng, 1000, 131072)
        prompts = _log(rng, 1, max(1, min(64, 32 * 16 * 131072 // 2 // (beams * vocab))))
        return _select(prompts, beams, vocab, min(64, 2 * beams + rng.randint(0, 3)), rng.choice(["fp32", "fp16", "bf16"]),
                       rng.random() < 0.5, rng.random() < 0.3)
    if kind == "pages":
        layers, kvh, head = rng.randint(1, 8), _log(rng, 1, 32), rng.choice([64, 72, 128, 160])
        pages = _log(rng, 16, 8 * 512 * 32 * 128 // (layers * kvh * head) // 4)
        return _pages(layers, kvh, pages, _log(rng, 1, min(1500, pages // 2 - 1)), head, rng.choice(["fp16", "bf16", "fp32"]),
                      rng.random() < 0.5)
    if kind == "states":
        beams = rng.randint(2, 8)
        return _states(rng.randint(1, 4), rng.randint(1, 16), rng.choice([48, 64, 128]), rng.choice([64, 96, 128]),
                       beams * rng.randint(1, 8), beams, rng.random() < 0.5)
    heads, kvh = rng.choice([(32, 32), (40, 40), (32, 8), (64, 8), (8, 1), (12, 3), (10, 5), (16, 16)])
    beams = rng.randint(1, 12)
    shared = _log(rng, 1, 1024) * BLOCK
    most = min(16, 16 * 8 * 32 * 2176 // (beams * kvh * (shared + 400)))
    return _attention(_log(rng, 1, max(1, most)), beams, heads, kvh, shared, _log(rng, 1, 400), rng.choice(["fp16", "bf16"]),
                      rng.random() < 0.5)


def prepare(case: dict, seed: int) -> dict:
    return _KINDS[case["kind"]][0](case, seed)


def run(state: dict):
    return _KINDS[state["c"]["kind"]][1](state)


def exact(case: dict, seed: int):
    return _KINDS[case["kind"]][2](prepare(case, seed))


def work(case: dict) -> dict:
    return _KINDS[case["kind"]][3](case)
