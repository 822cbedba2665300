"""Beam search through the engine against a search written down plainly, whose hypotheses share nothing: each one's whole
text is run as a prompt of its own at every step.

In 32 bits both searches see logits that differ by rounding alone and have to find the same hypotheses.  In 16 bits
near-equal candidates may change places: there every score found has to be the one that its tokens get when they are run
by themselves, and no best hypothesis worse than the plain search's but for that."""
import json

import pytest
import torch

from tests import buzalorn_util as B
from tests import movarax_util as M

pytestmark = pytest.mark.gpu


def small_llama(heads=4, kv=4, seed=0, vocab=384, max_seqs=12, kv_blocks=200, block=16, deltas=None):
    from deltazip_b200.engine import DecodeEngine
    from deltazip_b200.llama import LlamaConfig
    cfg = LlamaConfig(hidden_size=128 * heads, intermediate_size=512, num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv, vocab_size=vocab)
    torch.manual_seed(seed)
    eng = DecodeEngine(cfg, deltas, max_seqs, kv_blocks, block, seed=seed, dtype=torch.float16)
    with torch.no_grad():                          # weights that are more than noise behind the norms
        g = torch.Generator("cuda").manual_seed(seed + 1)
        for layer in eng.model.layers:
            for m in (layer.qkv_proj, layer.o_proj, layer.gate_up_proj, layer.down_proj):
                m.weight.normal_(0, 1.3 * m.weight.shape[1] ** -0.5, generator=g)
    return eng


def engine(kind, dtype=torch.float32, **kw):
    if kind == "buzalorn":
        config = B.make_config()
        return B.make_engine(config, B.make_tensors(config), dtype, **{**dict(max_seqs=12, kv_blocks=300), **kw})
    config = M.make_config()
    return M.make_engine(config, M.make_tensors(config), dtype, **{**dict(max_seqs=12, kv_blocks=300), **kw})


def log_probs(eng, texts, first, delta=0):
    """log-probabilities [tokens from `first` on of every text] of each next token, every text a sequence of its own."""
    from deltazip_b200.engine import Sequence
    out = []
    for i, text in enumerate(texts):
        seq = Sequence(1000 + i, delta, len(text), 0)
        assert eng.admit([seq])
        seq.length = 0
        with torch.inference_mode():
            h = eng.extend([(seq, text)])
            out.append(torch.log_softmax(eng.model.beam_logits(h[first - 1:]).double(), -1))
        eng.retire(seq)
    return out


def plain_search(eng, prompt, max_new, beams, stop_id=None, penalty=1.0, delta=0):
    live, ended = [([], 0.0)], []
    for step in range(1, max_new + 1):
        lp = [x[-1] for x in log_probs(eng, [prompt + t for t, _ in live], len(prompt), delta)]
        joint = torch.cat([x + s for x, (_, s) in zip(lp, live)])
        vocab = lp[0].numel()
        order = torch.sort(joint, descending=True, stable=True)[1][:2 * beams].tolist()
        nxt = []
        for rank, i in enumerate(order):
            if len(nxt) == beams:
                break
            text, score = live[i // vocab][0] + [i % vocab], float(joint[i])
            if i % vocab != stop_id:
                nxt.append((text, score))
            elif rank < beams:
                ended.append((text, score / len(text) ** penalty))
        live = nxt
    ended += [(t, s / len(t) ** penalty) for t, s in live]
    return sorted(ended, key=lambda e: -e[1])[:beams]


def prompts_of(lengths, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def through(eng):
    from deltazip_b200 import ops
    assert ops.read_status() == 0 and not eng.running and eng.cache.shared == 0
    assert sorted(eng.cache.free) == list(range(eng.cache.num_blocks)) and not any(eng.cache.holders)
    if eng.cache.state is not None:
        assert len(set(eng.cache.state.free)) == eng.cache.state.slots


@pytest.mark.parametrize("kind", ["buzalorn", "movarax"])
@pytest.mark.parametrize("beams,max_new,penalty", [(1, 6, 1.0), (4, 12, 1.0), (5, 9, 0.0), (3, 20, -0.5)])
def test_finds_what_a_plain_search_finds(kind, beams, max_new, penalty):
    """Layers with a window, matrix memories, latents and decays; more prompts than the batch holds at a time."""
    eng = engine(kind)
    prompts = prompts_of([1, 8, 19, 40, 7], 203, beams)
    got = eng.beam_search(prompts, max_new, beams, length_penalty=penalty)
    through(eng)
    for p, found in zip(prompts, got):
        want = plain_search(eng, p, max_new, beams, penalty=penalty)
        assert [h.tokens for h in found] == [t for t, _ in want]
        assert all(abs(h.score - s) <= 1e-4 * max(1, abs(s)) for h, (_, s) in zip(found, want))


@pytest.mark.parametrize("kind", ["buzalorn", "movarax"])
@pytest.mark.parametrize("penalty", [1.0, 0.0, 2.0])
def test_stop_token(kind, penalty):
    """Hypotheses end where the token comes; the search goes on until none can pass them."""
    eng = engine(kind)
    prompts = prompts_of([12, 5], 203, 3)
    free = eng.beam_search(prompts, 8, 4)
    stop = free[0][0].tokens[2]
    got = eng.beam_search(prompts, 8, 4, stop_id=stop, length_penalty=penalty)
    through(eng)
    if penalty <= 1:                               # (a larger one prefers what is long)
        assert any(h.tokens[-1] == stop and len(h.tokens) < 8 for h in got[0])
    for p, found in zip(prompts, got):
        want = plain_search(eng, p, 8, 4, stop, penalty)
        assert [h.tokens for h in found] == [t for t, _ in want]
        assert all(stop not in h.tokens[:-1] for h in found)


@pytest.mark.parametrize("heads,kv,block", [(4, 4, 16), (4, 1, 16), (4, 2, 5)])
def test_llama(heads, kv, block):
    eng = small_llama(heads, kv, block=block, kv_blocks=600)
    prompts = prompts_of([50, 3, 16, 33], 384, heads + kv)
    got = eng.beam_search(prompts, 10, 4)
    through(eng)
    for p, found in zip(prompts, got):
        assert len(found) == 4 and [h.score for h in found] == sorted((h.score for h in found), reverse=True)
        assert len({tuple(h.tokens) for h in found}) == 4
        for h in found:
            lp = log_probs(eng, [p + h.tokens[:-1]], len(p))[0]
            alone = sum(float(lp[i, t]) for i, t in enumerate(h.tokens)) / len(h.tokens)
            assert abs(alone - h.score) <= 0.02, (alone, h.score)
        want = plain_search(eng, p, 10, 4)
        assert found[0].score >= want[0][1] - 0.02


def test_llama_with_deltas():
    from deltazip_b200 import synth
    from deltazip_b200.config import DeltaConfig
    from deltazip_b200.models import DeltaModel
    eng = small_llama(deltas=DeltaConfig(max_deltas=2, max_bitwidth=4, max_cpu_deltas=4))
    gen = torch.Generator(device="cuda").manual_seed(1)
    for did in (1, 2, 3):
        tensors = {}
        for name, mod in eng.manager.modules.items():
            n, k = mod.weight.shape
            tensors[name] = synth.compress_delta_gptq(torch.randn((n, k), generator=gen, device="cuda") * 2e-2, 4)
        eng.manager.add_delta(DeltaModel.from_gptq_tensors(did, 4, tensors))
    prompts, deltas = prompts_of([20, 9, 31, 14], 384, 5), [2, 0, 1, 3]
    got = eng.beam_search(prompts, 6, 3, delta_ids=deltas)
    through(eng)
    for p, d, found in zip(prompts, deltas, got):
        assert len(found) == 3
        for h in found:
            lp = log_probs(eng, [p + h.tokens[:-1]], len(p), d)[0]
            alone = sum(float(lp[i, t]) for i, t in enumerate(h.tokens)) / len(h.tokens)
            assert abs(alone - h.score) <= 0.02, (d, alone, h.score)


def test_small_vocabulary():
    """Fewer tokens than hypotheses: what there is is continued."""
    config = M.make_config(vocab=5)
    eng = M.make_engine(config, M.make_tensors(config), torch.float32, max_seqs=9, kv_blocks=100)
    (got,) = eng.beam_search([[1, 4, 2]], 3, 9)
    through(eng)
    want = plain_search(eng, [1, 4, 2], 3, 9)
    assert [h.tokens for h in got] == [t for t, _ in want]
    (got,) = eng.beam_search([[1, 4, 2]], 1, 9)
    assert len(got) == 5


def test_greedy_is_a_search_with_one_hypothesis():
    eng = engine("movarax")
    prompts = prompts_of([9, 30], 203, 8)
    assert [f[0].tokens for f in eng.beam_search(prompts, 12, 1)] == eng.generate(prompts, 12)
    through(eng)


@pytest.mark.parametrize("kind", ["llama", "buzalorn", "movarax"])
def test_forks_decode_as_their_parents(kind):
    """A fork by hand, decoded greedily beside its parent and compacted on the way: the same tokens, from blocks and states
    of its own."""
    from deltazip_b200.engine import Sequence
    eng = small_llama() if kind == "llama" else engine(kind)
    prompt = prompts_of([37], 203, 2)[0]
    want = eng.generate([prompt], 14)[0]
    root = Sequence(0, 0, len(prompt), 20, prompt=torch.tensor(prompt))
    other = Sequence(1, 0, 5, 20, prompt=torch.tensor(prompt[:5]))
    assert len(eng.admit([other, root])) == 2
    eng.prefill([root, other])
    eng.retire(other)
    child = Sequence(5, 0, root.length, 20, generated=root.generated)
    eng.cache.fork([(root, child)])
    eng.running.append(child)
    first = {s: int(t) for s, t in zip([0, 1], eng.tokens.tolist())}[0]
    eng._rebuild({0: first, 5: first})
    got = [[first, first]]
    for step in range(13):
        got.append(eng.decode_step().tolist())
        if step == 6:
            used = eng.compact()
            assert used == len(set(root.blocks) | set(child.blocks)) == eng.cache.num_blocks - len(eng.cache.free)
    assert [g[0] for g in got] == want and [g[1] for g in got] == want
    for s in list(eng.running):
        eng.retire(s)
    through(eng)


def test_refusals():
    eng = engine("movarax", max_seqs=4, kv_blocks=6)
    for args in (([[1, 2]], 0, 2), ([[]], 3, 2), ([[1]], 3, 0), ([[1]], 3, 5)):
        with pytest.raises(ValueError):
            eng.beam_search(*args)
    with pytest.raises(RuntimeError):              # more blocks than there are
        eng.beam_search([list(range(40))], 20, 4)
    through(eng)
    assert len(eng.beam_search([[1, 2, 3]], 4, 3)[0]) == 3
    through(eng)


def test_command_line(tmp_path, capsys):
    from deltazip_b200.__main__ import main
    config = M.make_config()
    M.write_checkpoint(tmp_path, config, M.make_tensors(config))
    args = ["generate", "--model", str(tmp_path), "--prompt", "1 2 3", "--prompt", "9 8 7 6", "--max-new", "5", "--dtype", "float32"]
    assert main([*args, "--beams", "3", "--length-penalty", "0.5"]) == 0
    got = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    eng = engine("movarax")
    want = eng.beam_search([[1, 2, 3], [9, 8, 7, 6]], 5, 3, length_penalty=0.5)
    assert [[h["tokens"] for h in f] for f in got] == [[h.tokens for h in f] for f in want]
    assert main(args) == 0
    assert [json.loads(line) for line in capsys.readouterr().out.splitlines()] == eng.generate([[1, 2, 3], [9, 8, 7, 6]], 5)


@pytest.mark.parametrize("length", [5, 21, 32])
def test_one_hypothesis_that_forks_later(length, monkeypatch):
    """A step that leaves one candidate, and steps behind it that leave many: what the one hypothesis held is not taken for
    shared where its heirs write."""
    eng = small_llama(kv_blocks=600)
    prompts = prompts_of([length, length + 9], 384, length)
    plain, calls = eng.model.beam_logits, []

    def masked(hidden):
        logits = plain(hidden)
        calls.append(len(calls))
        if calls[-1] in (0, 1):
            logits = torch.full_like(logits, -float("inf"))
            logits[:, 5 + calls[-1]] = 0
        return logits
    monkeypatch.setattr(eng.model, "beam_logits", masked)
    got = eng.beam_search(prompts, 9, 4)
    monkeypatch.setattr(eng.model, "beam_logits", plain)
    through(eng)
    for p, found in zip(prompts, got):
        assert len(found) == 4 and len({tuple(h.tokens) for h in found}) == 4
        for h in found:
            assert h.tokens[:2] == [5, 6]
            lp = log_probs(eng, [p + h.tokens[:-1]], len(p))[0]
            alone = sum(float(lp[i, t]) for i, t in enumerate(h.tokens) if i > 1) / len(h.tokens)
            assert abs(alone - h.score) <= 0.02, (alone, h.score)
