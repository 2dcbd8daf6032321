"""Beam searches between ordinary requests of one engine, with decode graphs and without: what each gives does not depend on the others."""
import pytest
import torch

from mini_inference_b200 import BeamParams, SamplingParams
from tests.helpers import random_tokens
from tests.test_beam_search import TOL, check, engine


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["F", "W"])
def test_between_requests_of_an_engine_with_graphs(tiny_dirs, name, dtype):
    d, cfg, page = tiny_dirs[name]
    prompts = [random_tokens(cfg["vocab_size"], n, seed=n) for n in (9, 2 * page + 1, 4)]
    greedy, beams = SamplingParams(max_new_tokens=page + 6, ignore_eos=True), BeamParams(num_beams=3, max_new_tokens=page + 2, ignore_eos=True)
    plain = engine(d, page, "cuda:0", dtype=dtype)
    want_beams, want = plain.beam_search(prompts, beams), plain.generate(prompts, greedy)
    llm = engine(d, page, "cuda:0", dtype=dtype, cuda_graphs=True)
    for _ in range(2):
        # (float32 graphs and eager steps may sum products in different orders; the searches run the same steps)
        first = llm.generate(prompts, greedy)
        got = llm.beam_search(prompts, beams)
        assert [[(b.tokens, b.score) for b in bs] for bs in got] == [[(b.tokens, b.score) for b in bs] for bs in llm.beam_search(prompts, beams)]
        assert llm.generate(prompts, greedy) == first
        llm.cache.check_invariants()
        if dtype == "float32":
            assert first == want and [[b.tokens for b in bs] for bs in got] == [[b.tokens for b in bs] for bs in want_beams]
    if dtype == "float32":
        check(llm, prompts, beams, TOL)
    torch.cuda.synchronize()
