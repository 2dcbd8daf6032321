"""Beam search's running scores over long searches: sums of log-probabilities in 64 bits, and the order of beams that lie close together."""
import math

import pytest
import torch

from mini_inference_b200 import BeamParams
from mini_inference_b200.engine.beam import BeamGroup, BeamSearch
from tests.helpers import random_tokens
from tests.ref_beam import BeamRefOps
from tests.test_beam_search import engine

DEV = "cuda:0"


def search_on(device):
    search = BeamSearch.__new__(BeamSearch)
    if device == "cpu":
        search.ops = BeamRefOps()
    else:
        from mini_inference_b200.ops import get_ops
        search.ops = get_ops(device)
    return search


DEVICES = ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_beams_closer_than_a_long_score_rounds(device):
    """A score of -800 in float32 is off by up to 3e-5; beams 1e-5 apart stay in their order, whatever order they stand in."""
    search = search_on(device)
    for order in ([0, 1, 2, 3], [3, 1, 0, 2], [2, 3, 1, 0]):
        g = BeamGroup([1], BeamParams(num_beams=4, max_new_tokens=2000, ignore_eos=True), set())
        g.tokens, g.scores = [[7]] * 4, [-800.0 - 1e-5 * i for i in order]
        logits = torch.zeros(4, 50, device=device)
        logits[:, 9] = 30.0                                        # the same for all, and certain: -4.6e-12 from here
        (_, parents), = search._select([g], logits)
        assert parents == [order.index(i) for i in range(4)]
        assert all(abs(s + 800.0 + 1e-5 * i) < 1e-9 for i, s in enumerate(g.scores))


@pytest.mark.parametrize("device", DEVICES)
def test_long_sums(device):
    """300 steps of five beams.  A step rounds two numbers to float32, what a beam is behind its prompt's best one and the candidate's value, both below 16 here: half a step
    is 2^-21.  A running score in float32 would add half a step of its own size, 2^-16 from 256 on and 2^-15 from 512 on, in every one."""
    search, n, V, steps = search_on(device), 5, 40, 300
    gen = torch.Generator().manual_seed(1)
    table = torch.randn(V, V, generator=gen)                       # logits behind each token
    g = BeamGroup([1], BeamParams(num_beams=n, max_new_tokens=2 * steps, ignore_eos=True), set())
    g.tokens, g.scores = [[1]], [0.0]
    log_p = torch.log_softmax(table.double(), -1)
    for step in range(steps):
        ends = [t[-1] for t in g.tokens]
        search._select([g], table[ends].contiguous().to(device))
    assert min(g.scores) < -500 and not g.done
    for tokens, score in zip(g.tokens, g.scores):
        want = sum(float(log_p[a, b]) for a, b in zip(tokens, tokens[1:]))
        assert abs(score - want) <= steps * (2.0 ** -20 + 1e-8)
    assert g.scores == sorted(g.scores, reverse=True) and all(math.isfinite(s) for s in g.scores)


def test_the_engine_s_scores(tiny_dirs):
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, "cpu")
    prompt = random_tokens(256, 5, seed=4)
    beams = llm.beam_search([prompt], BeamParams(num_beams=3, max_new_tokens=60, ignore_eos=True))[0]
    for b in beams:
        lp = torch.log_softmax(llm.score(prompt + b.tokens).double(), -1)
        want = sum(float(lp[len(prompt) - 1 + i, t]) for i, t in enumerate(b.tokens))
        assert abs(b.score - want) <= 60 * (2.0 ** -20 + 1e-5)     # (a step's logits and the whole hypothesis' agree to 1e-5 or so)


def test_lengths_whose_power_is_no_number_are_refused():
    """A rank divides by a length to the power of length_penalty."""
    for n, p in ((100000, 64.0), (100000, -64.0), (2 ** 31, 40.0), (10 ** 300, 1.5)):
        with pytest.raises(ValueError, match="length_penalty"):
            BeamParams(max_new_tokens=n, length_penalty=p)
    for n, p in ((10000, 64.0), (10000, -64.0), (2 ** 20, 40.0), (2 ** 40, 1.0), (1, 64.0)):
        g = BeamGroup([1], BeamParams(max_new_tokens=n, length_penalty=p, num_beams=1), {7})
        g.tokens = [[3] * (n - 1 if n < 2 ** 21 else 10)]
        g.advance([(-1e4, 0, 7)])
        assert math.isfinite(g.ended[0].rank) and g.ended[0].rank < 0
