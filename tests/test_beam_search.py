"""Beam search through the engine: against a search that scores every hypothesis from its first token on (no shared pages, no states taken over), for every
architecture, on the CPU with plain kernel statements and on the GPU with the kernels; the cache's forks and takeovers; host bookkeeping."""
import importlib
import math
import random

import pytest
import torch

from mini_inference_b200 import LLM, Beam, BeamParams, SamplingParams
from mini_inference_b200.cache import CacheManager
from mini_inference_b200.engine.beam import BeamGroup
from mini_inference_b200.engine.runner import CacheFull
from mini_inference_b200.parts.base import KVCacheNeed, StateNeed
from mini_inference_b200.weights import write_random_model
from tests.conftest import TINY
from tests.helpers import random_tokens
from tests.ref_beam import BeamRefOps

gpu = pytest.mark.gpu


# ---------------------------------------------------------------- a search without any sharing
def plain_search(llm, prompt, params):
    """The same search in its plain form: every step scores all live hypotheses whole, by llm.score, in 64 bits."""
    n, eos = params.num_beams, set() if params.ignore_eos else llm.eos_ids
    live, ended = [(0.0, [])], []
    rank = lambda s, t: s / len(t) ** params.length_penalty       # noqa: E731
    while True:
        found = []
        for b, (s, toks) in enumerate(live):
            lp = torch.log_softmax(llm.score(prompt + toks)[-1].double().cpu(), 0)
            top = torch.sort(lp, descending=True, stable=True).indices[:2 * n].tolist()
            found += [(s + float(lp[t]), b, t) for t in top]
        found.sort(key=lambda f: (-f[0], f[1]))
        nxt = []
        for i, (s, b, t) in enumerate(found[:2 * n]):
            if t in eos:
                if i < n:
                    ended.append((rank(s, live[b][1] + [t]), s, live[b][1] + [t], "stop"))
            elif len(nxt) < n:
                nxt.append((s, live[b][1] + [t]))
        ended = sorted(ended, key=lambda e: -e[0])[:n]
        live = nxt
        length = len(live[0][1]) if live else params.max_new_tokens
        if length >= params.max_new_tokens:
            return sorted(ended + [(rank(s, t), s, t, "length") for s, t in live], key=lambda e: -e[0])[:n]
        if len(ended) == n:
            p = params.length_penalty
            if live[0][0] / (length if p <= 0 else params.max_new_tokens) ** p <= ended[-1][0]:
                return ended


def check(llm, prompts, params, tol):
    pool, slots = llm.cache.free_pages(), llm.cache.slots.num_free
    got = llm.beam_search(prompts, params)
    llm.cache.check_invariants()
    assert (llm.cache.free_pages(), llm.cache.slots.num_free) == (pool, slots)
    assert len(got) == len(prompts)
    for prompt, beams in zip(prompts, got):
        want = plain_search(llm, prompt, params)
        assert len(beams) == len(want) and all(isinstance(b, Beam) for b in beams)
        for b, (rank, score, tokens, reason) in zip(beams, want):
            assert abs(b.rank - rank) <= tol * (1 + abs(rank)), (b, rank, tokens)
            assert (b.tokens, b.finish_reason) == (tokens, reason), (b, rank, tokens)
            assert abs(b.score - score) <= tol * (1 + abs(score))
        assert [b.rank for b in beams] == sorted((b.rank for b in beams), reverse=True)


def engine(d, page, device, **kw):
    ops = BeamRefOps() if device == "cpu" else None
    return LLM(d, dtype=kw.pop("dtype", "float32"), device=device, ops=ops, **{**dict(kv_block_size=page, kv_cache_tokens=2048, max_num_seqs=12), **kw})


DEVICES = ["cpu", pytest.param("cuda:0", marks=gpu)]
# float32 steps of one, two and more rows sum in different orders: their logits agree to 1e-5 or so, a hypothesis adds those of its tokens
TOL = 2e-4


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["A", "B", "W", "F", "V"])
def test_against_a_search_without_sharing(tiny_dirs, name, device):
    d, cfg, page = tiny_dirs[name]
    llm = engine(d, page, device)
    prompts = [random_tokens(cfg["vocab_size"], n, seed=n) for n in (5, page, 2 * page + 1)]
    check(llm, prompts, BeamParams(num_beams=4, max_new_tokens=2 * page + 3, ignore_eos=True), TOL)
    check(llm, prompts[:1], BeamParams(num_beams=1, max_new_tokens=5, ignore_eos=True), TOL)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("design", ["naditar", "namesun", "nununex", "megovik", "fetodra", "kofutar"])
def test_designs_with_states_and_windows(tmp_path_factory, design, device):
    """Recurrent states, filters' last inputs, windows, latent rows, borrowed keys: whatever a design keeps moves with its beam."""
    tests = importlib.import_module("tests.test_" + design)
    for i, name in enumerate(sorted(tests.CONFIGS)):
        cfg, page = tests.CONFIGS[name]
        d = str(tmp_path_factory.mktemp(f"beam_{design}_{name}"))
        write_random_model(cfg, d, seed=30 + i, std=getattr(tests, "STD", 0.1), norm_init="uniform")
        llm = engine(d, page, device)
        prompts = [random_tokens(llm.model.spec.vocab_size, n, seed=n + i) for n in (4, page + 3)]
        check(llm, prompts, BeamParams(num_beams=3, max_new_tokens=page + 4, ignore_eos=True), TOL)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("penalty", [1.0, 0.0, 2.5, -1.0])
def test_ends_of_sequence_and_length_penalty(tiny_dirs, penalty, device):
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, device)
    prompts = [random_tokens(256, n, seed=n) for n in (7, 12, 3)]
    # tokens that the search meets anyway end it
    free = llm.beam_search(prompts, BeamParams(num_beams=4, max_new_tokens=12, ignore_eos=True))
    llm.eos_ids = {free[0][0].tokens[3], free[1][1].tokens[5], free[2][3].tokens[1], free[2][0].tokens[6]}
    check(llm, prompts, BeamParams(num_beams=4, max_new_tokens=12, length_penalty=penalty), TOL)
    check(llm, prompts, BeamParams(num_beams=2, max_new_tokens=1, length_penalty=penalty), TOL)


@pytest.mark.parametrize("device", DEVICES)
def test_prompts_in_waves_and_in_portions(tiny_dirs, device):
    """More prompts than there are slots, and prompts longer than a step's budget."""
    d, cfg, page = tiny_dirs["F"]
    llm = engine(d, page, device, max_num_seqs=7, max_batched_tokens=16)
    prompts = [random_tokens(cfg["vocab_size"], n, seed=n) for n in (40, 3, 16, 17, 33)]
    check(llm, prompts, BeamParams(num_beams=3, max_new_tokens=6, ignore_eos=True), TOL)
    tight = engine(d, page, device, max_num_seqs=8, kv_cache_tokens=page * 15, kv_watermark=0.0)
    check(tight, prompts[1:4], BeamParams(num_beams=4, max_new_tokens=5, ignore_eos=True), TOL)


@pytest.mark.parametrize("device", DEVICES)
def test_more_beams_than_continuations(tmp_path_factory, device):
    """A vocabulary smaller than twice the beams."""
    cfg = dict(TINY["A"][0], vocab_size=5)
    d = str(tmp_path_factory.mktemp("five"))
    write_random_model(cfg, d, seed=3, std=0.3, norm_init="uniform")
    llm = engine(d, 4, device)
    got = llm.beam_search([[1, 2], [4]], BeamParams(num_beams=9, max_new_tokens=3, ignore_eos=True))
    for prompt, beams in zip(([1, 2], [4]), got):
        assert len(beams) == 9 and len({tuple(b.tokens) for b in beams}) == 9
        for b in beams:
            lp = torch.log_softmax(llm.score(prompt + b.tokens).double().cpu(), -1)
            want = sum(float(lp[len(prompt) - 1 + i, t]) for i, t in enumerate(b.tokens))
            assert abs(b.score - want) < TOL * (1 + abs(want))
    llm.cache.check_invariants()


def test_greedy_is_one_beam(tiny_dirs):
    d, cfg, page = tiny_dirs["B"]
    llm = engine(d, page, "cpu")
    prompt = random_tokens(cfg["vocab_size"], 9, seed=1)
    one = llm.beam_search([prompt], BeamParams(num_beams=1, max_new_tokens=8, ignore_eos=True))[0][0]
    assert one.tokens == llm.generate([prompt], SamplingParams(max_new_tokens=8, ignore_eos=True))[0]


def test_refusals(tiny_dirs):
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, "cpu", max_num_seqs=4, kv_cache_tokens=page * 8, kv_watermark=0.0)
    for bad in (dict(num_beams=0), dict(num_beams=65), dict(max_new_tokens=0), dict(length_penalty=math.nan), dict(length_penalty=math.inf), dict(length_penalty=65.0), dict(length_penalty=-1e9)):
        with pytest.raises(ValueError):
            BeamParams(**bad)
    with pytest.raises(ValueError, match="holds 4 sequences"):
        llm.beam_search([[1, 2]], BeamParams(num_beams=5, max_new_tokens=2))
    with pytest.raises(ValueError, match="empty"):
        llm.beam_search([[]], BeamParams(num_beams=2, max_new_tokens=2))
    with pytest.raises(ValueError, match="token id"):
        llm.beam_search([[1], [256]], BeamParams(num_beams=2, max_new_tokens=2))
    with pytest.raises(ValueError, match="limit"):
        llm.beam_search([[1] * 60], BeamParams(num_beams=2, max_new_tokens=10))
    with pytest.raises(CacheFull):
        llm.beam_search([[1] * 40], BeamParams(num_beams=4, max_new_tokens=20))
    llm.add_request([1, 2, 3], SamplingParams(max_new_tokens=2))
    with pytest.raises(RuntimeError, match="by itself"):
        llm.beam_search([[1]], BeamParams(num_beams=2, max_new_tokens=2))
    while llm.has_work():
        llm.step()
    assert llm.beam_search([], BeamParams(num_beams=2, max_new_tokens=2)) == []
    llm.cache.check_invariants()
    assert llm.cache.free_pages() == 8 and llm.cache.slots.num_free == 4


def test_a_failed_step_gives_everything_back(tiny_dirs, monkeypatch):
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, "cpu")
    pool, calls, inner = llm.cache.free_pages(), [], llm.runner.step

    def failing(*a, **kw):
        calls.append(1)
        if len(calls) == 5:
            raise RuntimeError("lost")
        return inner(*a, **kw)
    monkeypatch.setattr(llm.runner, "step", failing)
    with pytest.raises(RuntimeError, match="lost"):
        llm.beam_search([[1, 2, 3], [4]], BeamParams(num_beams=3, max_new_tokens=9, ignore_eos=True))
    llm.cache.check_invariants()
    assert llm.cache.free_pages() == pool and llm.cache.slots.num_free == 12
    monkeypatch.undo()
    check(llm, [[1, 2, 3], [4]], BeamParams(num_beams=3, max_new_tokens=4, ignore_eos=True), TOL)


# ---------------------------------------------------------------- the cache
NEEDS = [KVCacheNeed(2, 8), KVCacheNeed(2, 8, window=11, keep_first=5), (KVCacheNeed(1, 6, planes=1), StateNeed((3, 5))), KVCacheNeed(2, 8, value_dim=4), StateNeed((7,), "int32"),
         StateNeed((9,), "compute"), KVCacheNeed(2, 8)]


def content(cache, seq):
    """What a request's cache holds: its cached tokens' rows of every group, and its states."""
    out = []
    for gi, g in enumerate(cache.kv_groups):
        live = [i for i in range(seq.num_tokens) if i // cache.page_size in set(cache._live_pages(gi, seq))]
        at = cache.slots_for(gi, seq, 0, seq.num_tokens)[live]
        page, off = torch.as_tensor(at // cache.page_size).long(), torch.as_tensor(at % cache.page_size).long()
        out.append(g.storage[:, :, page, :, off].clone())
        if g.value_storage is not None:
            out.append(g.value_storage[:, page, :, off].clone())
    return out + [g.storage[seq.slot].clone() for g in cache.state_groups]


def write(cache, seq, start, end, rng):
    for gi, g in enumerate(cache.kv_groups):
        for at in cache.slots_for(gi, seq, start, end).tolist():
            page, off = divmod(at, cache.page_size)
            g.storage[:, :, page, :, off] = torch.rand(g.storage[:, :, page, :, off].shape, generator=rng).to(g.storage)
            if g.value_storage is not None:
                g.value_storage[:, page, :, off] = torch.rand(g.value_storage[:, page, :, off].shape, generator=rng).to(g.value_storage)
    for g in cache.state_groups:
        g.storage[seq.slot] = (torch.rand(g.storage[seq.slot].shape, generator=rng) * 1000).to(g.storage)


@pytest.mark.parametrize("device", DEVICES)
def test_forks_and_takeovers(device):
    """Random prompts, beams and parents: every beam holds what its parent held, whatever was shared, in every group and state; nothing leaks."""
    if device == "cpu":
        ops = BeamRefOps()
    else:
        from mini_inference_b200.ops import get_ops
        ops = get_ops(device)
    rng, gen = random.Random(4), torch.Generator().manual_seed(4)
    cache = CacheManager(NEEDS, 4, 120, 10, 64, dtype=torch.float32, device=device)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))       # noqa: E731
    for turn in range(12):
        families = []
        for f in range(2):
            n, length = rng.choice([1, 2, 4, 5]), rng.choice([1, 3, 4, 5, 8, 13])
            seq = cache.admit((turn, f, 0))
            assert cache.ensure(seq, length)
            write(cache, seq, 0, length, gen)
            cache.commit(seq, length)
            held = content(cache, seq)
            seqs = [seq] + cache.fork(seq, [(turn, f, i) for i in range(1, n)])
            families.append((seqs, [held] + [None] * (n - 1)))
        cache.reorder([(seqs, [0] * len(seqs)) for seqs, _ in families], ops)
        families = [(seqs, [held[0]] * len(seqs)) for seqs, held in families]
        for step in range(rng.randint(1, 14)):
            moves = []
            for k, (seqs, held) in enumerate(families):
                assert all(same(content(cache, s), h) for s, h in zip(seqs, held))
                for s in seqs:
                    n = s.num_tokens
                    assert cache.ensure(s, n + 1)
                    write(cache, s, n, n + 1, gen)
                    cache.commit(s, n + 1)
                held = [content(cache, s) for s in seqs]
                parents = [rng.randrange(len(seqs)) for _ in seqs] if rng.random() < 0.8 else list(range(len(seqs)))
                moves.append((seqs, parents))
                families[k] = (seqs, [held[p] for p in parents])
            cache.reorder(moves, ops)
            if device != "cpu":
                for gi in range(len(cache.kv_groups)):
                    idx, val = cache.take_table_updates(gi)
                    ops.scatter_i32(cache.kv_groups[gi].device_table.view(-1), torch.tensor(idx, device=device), torch.tensor(val, device=device))
            cache.check_invariants()
            for seqs, _ in families:
                s0, shared = seqs[0], seqs[0].family.shared if len(seqs) > 1 else 0
                pages = shared // cache.page_size
                assert all((cache.kv_groups[0].tables[s.slot, :pages] == cache.kv_groups[0].tables[s0.slot, :pages]).all() for s in seqs)
        for seqs, _ in families:
            for s in rng.sample(seqs, len(seqs)):
                cache.free(s)
                cache.check_invariants()
        assert all(g.pool.num_free == 120 and not any(g.pool.ref) for g in cache.kv_groups) and cache.slots.num_free == 10


def test_fork_takes_nothing_where_something_is_short():
    cache = CacheManager([KVCacheNeed(1, 8)], 4, 6, 4, 64, dtype=torch.float32)
    a = cache.admit("a")
    cache.ensure(a, 14)
    cache.commit(a, 14)                                   # four pages of six
    assert cache.fork(a, ["b", "c", "d"]) is None         # three last pages, two are free
    assert cache.fork(a, ["b", "c", "d", "e"]) is None    # four slots, three are free
    assert cache.free_pages() == 2 and cache.slots.num_free == 3
    b, c = cache.fork(a, ["b", "c"])
    assert cache.free_pages() == 0 and a.family.shared == 12
    with pytest.raises(RuntimeError):
        cache.fork(a, ["b"])
    with pytest.raises(ValueError):
        cache.reorder([([a, b, c], [0, 3, 1])], BeamRefOps())
    d = cache.admit("d")
    with pytest.raises(RuntimeError):
        cache.reorder([([a, d], [0, 0])], BeamRefOps())
    for s in (b, a, d, c):
        cache.free(s)
    cache.check_invariants()
    assert cache.free_pages() == 6


# ---------------------------------------------------------------- bookkeeping
def test_endings_beyond_the_best_do_not_count():
    g = BeamGroup([1], BeamParams(num_beams=2, max_new_tokens=9, length_penalty=0.0), {7})
    assert g.advance([(-1.0, 0, 3), (-2.0, 0, 4), (-3.0, 0, 7), (-4.0, 0, 5)]) == [0, 0]
    assert g.tokens == [[3], [4]] and g.scores == [-1.0, -2.0] and not g.ended
    assert g.advance([(-1.5, 0, 7), (-2.5, 1, 6), (-2.6, 0, 8), (-9.0, 1, 1)]) == [1, 0]
    assert [b.tokens for b in g.ended] == [[3, 7]] and g.tokens == [[4, 6], [3, 8]] and not g.done
    assert g.advance([(-2.6, 0, 7), (-2.7, 1, 7), (-3.0, 1, 2), (-4.0, 0, 2)]) == [1, 0]
    assert [b.score for b in g.ended] == [-1.5, -2.6] and g.done       # what goes on has -3 and falls


def test_groups_without_continuations_end():
    g = BeamGroup([1], BeamParams(num_beams=2, max_new_tokens=9), {7})
    g.advance([(-1.0, 0, 3)])
    assert g.scores == [-1.0, -math.inf] and not g.done
    g.advance([(-1.25, 0, 7)])
    assert g.done and [b.tokens for b in g.ended] == [[3, 7]] and g.ended[0].finish_reason == "stop"
