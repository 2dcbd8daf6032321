"""What beams are said to share (Family.shared), on the CPU: never more than lies on the same pages in all of a prompt's beams, whichever of them forked or were reordered last."""
import random

import pytest
import torch

from mini_inference_b200.cache import CacheManager
from mini_inference_b200.engine.batch import shared_of
from mini_inference_b200.parts.base import KVCacheNeed, StateNeed
from tests.ref_beam import BeamRefOps

PS = 4


def cache_of(pages=200):
    return CacheManager([KVCacheNeed(2, 8), StateNeed((3,)), KVCacheNeed(1, 8, window=9)], PS, pages, 16, 80, dtype=torch.float32)


def grow(cache, seqs, n):
    for s in seqs:
        assert cache.ensure(s, s.num_tokens + n)
        cache.commit(s, s.num_tokens + n)


def check(cache, seqs):
    """All living beams read the first one's pages for the keys that they are said to share."""
    shared = {n for _, n in shared_of(seqs, [1] * len(seqs))}
    assert len(shared) == 1
    pages, rest = divmod(shared.pop(), PS)
    tables = cache.kv_groups[0].tables[[s.slot for s in seqs]]
    assert not rest and pages <= min(s.num_tokens for s in seqs) // PS and (tables[:, :pages] == tables[0, :pages]).all()
    cache.check_invariants()
    return pages


def family(n=3, length=6):
    cache = cache_of()
    a = cache.admit("a")
    assert cache.ensure(a, length)
    cache.commit(a, length)
    seqs = [a] + cache.fork(a, [f"a{i}" for i in range(1, n)])
    cache.reorder([(seqs, [0] * n)], BeamRefOps())
    return cache, seqs


def test_a_beam_that_forks_again():
    cache, seqs = family()
    assert check(cache, seqs) == 1
    grow(cache, seqs, 9)                                          # pages of their own
    seqs += cache.fork(seqs[1], ["b"])
    assert check(cache, seqs) == 1                                # "b" has more in common with one of them, not with all


def test_some_of_the_beams_reordered():
    cache, seqs = family(4)
    grow(cache, seqs, 9)
    cache.reorder([(seqs[:2], [1, 1])], BeamRefOps())
    assert check(cache, seqs) == 1
    cache.reorder([(seqs, [2, 2, 2, 2])], BeamRefOps())
    assert check(cache, seqs) == 15 // PS


def test_beams_that_are_given_up():
    cache, seqs = family(4)
    grow(cache, seqs, 9)
    cache.reorder([(seqs[:3], [1, 1, 1])], BeamRefOps())
    assert check(cache, seqs) == 1
    cache.free(seqs.pop())                                        # what is left shares more, and may be said to
    assert 1 <= check(cache, seqs) <= 15 // PS
    for s in seqs[1:]:
        cache.free(s)
    check(cache, seqs[:1])


@pytest.mark.parametrize("seed", range(6))
def test_at_random(seed):
    rng, ops = random.Random(seed), BeamRefOps()
    cache, seqs = family(rng.randint(1, 4), rng.randint(1, 14))
    for turn in range(40):
        what = rng.random()
        if what < 0.4:
            grow(cache, seqs, rng.randint(1, 3)) if max(s.num_tokens for s in seqs) < 70 else None
        elif what < 0.55 and len(seqs) < 8:
            parent = rng.choice(seqs)
            child, = cache.fork(parent, [(turn, "child")])
            seqs.append(child)
            cache.reorder([([parent, child], [0, 0])], ops)
        elif what < 0.85:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            cache.reorder([(some, [rng.randrange(len(some)) for _ in some])], ops)
        elif len(seqs) > 1:
            cache.free(seqs.pop(rng.randrange(len(seqs))))
        check(cache, seqs)


class NoMoreThanFour(BeamRefOps):
    MAX_BEAMS = 4

    def reorder_rows(self, tensors, rows, parents, group_start, most, dim=0):
        assert most <= 4
        super().reorder_rows(tensors, rows, parents, group_start, most, dim)


def test_a_refused_group_changes_nothing():
    """... of the groups in front of it either."""
    cache, seqs = family(4, 9)
    grow(cache, seqs, 6)
    other = cache.admit("other")
    assert cache.ensure(other, 15)
    cache.commit(other, 15)
    more = [other] + cache.fork(other, [f"o{i}" for i in range(1, 6)])
    before = [g.tables.copy() for g in cache.kv_groups], [list(g.pool.ref) for g in cache.kv_groups]
    for bad, error in (([(seqs, [1, 1, 0, 0]), (more[:2], [0, 2])], ValueError), ([(seqs, [1, 1, 0, 0]), (more[:2], [0])], ValueError),
                       ([(seqs, [1, 1, 0, 0]), ([other, seqs[0]], [0, 0])], RuntimeError), ([(seqs, [1, 1, 0, 0]), (more, [0] * 6)], ValueError),
                       ([(seqs[:2], [1, 1]), (seqs[1:], [0, 0, 0])], RuntimeError), ([([seqs[0], seqs[0]], [1, 1])], RuntimeError)):
        with pytest.raises(error):
            cache.reorder(bad, NoMoreThanFour())
        assert all((a == g.tables).all() for a, g in zip(before[0], cache.kv_groups)) and before[1] == [list(g.pool.ref) for g in cache.kv_groups]
        cache.check_invariants()
    cache.reorder(iter([(seqs, [1, 1, 0, 0]), (more[:4], [1, 1, 0, 0])]), NoMoreThanFour())
    check(cache, seqs)


def test_a_cache_without_storage():
    """Tables and pages alone."""
    cache = CacheManager([KVCacheNeed(2, 8), StateNeed((3,))], PS, 40, 8, 80, dtype=torch.float32, allocate=False)
    a = cache.admit("a")
    assert cache.ensure(a, 6)
    cache.commit(a, 6)
    seqs = [a] + cache.fork(a, ["b", "c"])
    cache.reorder([(seqs, [0, 0, 0])], BeamRefOps())
    grow(cache, seqs, 7)
    cache.reorder([(seqs, [2, 2, 0])], BeamRefOps())
    check(cache, seqs)
