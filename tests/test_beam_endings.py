"""Beam search with several end tokens: against a search that looks at every candidate of the vocabulary in every step."""
import pytest
import torch

from mini_inference_b200 import BeamParams
from mini_inference_b200.engine.beam import BeamGroup, BeamSearch
from tests.helpers import random_tokens
from tests.ref_beam import BeamRefOps
from tests.test_beam_search import DEVICES, TOL, engine


def search_all(llm, prompt, params):
    """Every hypothesis scored whole by llm.score, every token a candidate: the n best that do not end go on, endings count among the n best of all."""
    n, eos, p = params.num_beams, llm.eos_ids, params.length_penalty
    live, ended = [(0.0, [])], []
    rank = lambda s, t: s / len(t) ** p                           # noqa: E731
    while True:
        found = []
        for b, (s, toks) in enumerate(live):
            lp = torch.log_softmax(llm.score(prompt + toks)[-1].double().cpu(), 0)
            found += [(-(s + x), b, t) for t, x in enumerate(lp.tolist())]
        found.sort()
        for s, b, t in found[:n]:
            if t in eos:
                ended.append((rank(-s, live[b][1] + [t]), -s, live[b][1] + [t], "stop"))
        live = [(-s, live[b][1] + [t]) for s, b, t in found if t not in eos][:n]
        ended = sorted(ended, key=lambda e: -e[0])[:n]
        length = len(live[0][1])
        if length >= params.max_new_tokens:
            return sorted(ended + [(rank(s, t), s, t, "length") for s, t in live], key=lambda e: -e[0])[:n]
        if len(ended) == n and live[0][0] / (length if p <= 0 else params.max_new_tokens) ** p <= ended[-1][0]:
            return ended


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("ends", [1, 3, 9, 60])
@pytest.mark.parametrize("beams,penalty", [(2, 1.0), (4, 0.0), (5, 2.5)])
def test_several_end_tokens(tiny_dirs, beams, penalty, ends, device):
    """Up to all of a step's best candidates end.  60 end tokens are more than all of a prompt's candidates together leave room for."""
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, device)
    prompts = [random_tokens(256, n, seed=n) for n in (7, 12, 3)]
    llm.eos_ids = set(llm.score(prompts[0])[-1].argsort(descending=True)[:ends].tolist())      # what the first prompt's search would choose first
    params = BeamParams(num_beams=beams, max_new_tokens=7, length_penalty=penalty)
    for prompt, got in zip(prompts, llm.beam_search(prompts, params)):
        want = search_all(llm, prompt, params)
        assert [(b.tokens, b.finish_reason) for b in got] == [(t, reason) for _, _, t, reason in want]
        assert all(abs(b.score - s) <= TOL * (1 + abs(s)) for b, (_, s, _, _) in zip(got, want))
    llm.cache.check_invariants()


@pytest.mark.parametrize("device", DEVICES)
def test_more_candidates_than_the_selection_gives(tiny_dirs, device):
    """33 beams and 3 end tokens: 132 candidates may be needed, 128 come; they are selected row by row instead."""
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, device, max_num_seqs=40)
    prompt = random_tokens(256, 6, seed=2)
    first = llm.score(prompt)[-1].argsort(descending=True)[:3].tolist()
    llm.eos_ids = set(first)
    params = BeamParams(num_beams=33, max_new_tokens=3, length_penalty=0.0)
    got, want = llm.beam_search([prompt], params)[0], search_all(llm, prompt, params)
    assert [(b.tokens, b.finish_reason) for b in got] == [(t, reason) for _, _, t, reason in want]


def test_more_end_tokens_than_can_be_looked_past(tiny_dirs):
    d, cfg, page = tiny_dirs["A"]
    llm = engine(d, page, "cpu", max_num_seqs=64)
    llm.eos_ids = set(range(65))
    with pytest.raises(ValueError, match="end-of-sequence tokens"):
        llm.beam_search([[1, 2]], BeamParams(num_beams=64, max_new_tokens=2))
    assert len(llm.beam_search([[1, 2]], BeamParams(num_beams=4, max_new_tokens=2))[0]) == 4
    assert len(llm.beam_search([[1, 2]], BeamParams(num_beams=64, max_new_tokens=2, ignore_eos=True))[0]) == 64
    llm.eos_ids = set(range(1000, 2000)) | {3}                     # tokens that the vocabulary does not have end nothing
    assert len(llm.beam_search([[1, 2]], BeamParams(num_beams=64, max_new_tokens=2))[0]) == 64


class Asked(BeamRefOps):
    def beam_select(self, logits, scores, group_start, num):
        self.num = num
        assert num <= 128
        return super().beam_select(logits, scores, group_start, num)


@pytest.mark.parametrize("ends", [{7}, {7, 8}, {7, 8, 9, 10, 11}, set(range(5, 100))])
def test_enough_candidates_to_go_on(ends):
    """The best candidates all end; as many beams go on as there are."""
    ops = Asked()
    search = BeamSearch.__new__(BeamSearch)
    search.ops = ops
    for n in (2, 3, 20):
        g = BeamGroup([1], BeamParams(num_beams=n, max_new_tokens=9), ends)
        g.tokens, g.scores = [[3]] * n, [-1.0 - 0.01 * i for i in range(n)]
        logits = torch.randn(n, 200, generator=torch.Generator().manual_seed(n))
        logits[:, list(ends)] += 20.0
        (_, parents), = search._select([g], logits)
        assert len(parents) == n and all(s > -1e30 for s in g.scores) and not {t[-1] for t in g.tokens} & ends
        assert len(g.ended) == n
        lp = torch.log_softmax(logits.double(), -1) + torch.tensor([-1.0 - 0.01 * i for i in range(n)], dtype=torch.float64)[:, None]
        lp[:, list(ends)] = -1e30
        best = lp.flatten().sort(descending=True).indices[:n].tolist()
        assert [(p, t[-1]) for p, t in zip(parents, g.tokens)] == [divmod(i, 200) for i in best]
