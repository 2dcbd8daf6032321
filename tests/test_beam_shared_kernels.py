"""The kernels that share prefixes, reached through LLM.beam_search: whole searches against one without any sharing, and every single call against 64 bits by each row's own
pages, so that a wrong group or a prefix said too long shows."""
import types

import pytest
import torch

from mini_inference_b200 import BeamParams
from mini_inference_b200.ops import CudaOps
from mini_inference_b200.weights import write_random_model
from tests.conftest import TINY
from tests.helpers import random_tokens
from tests.ref_beam import shared_prefix_attention64
from tests.test_beam_search import TOL, check, engine

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
# heads of 64 in groups of 3, pages of 16 (also with windowed layers between), and heads of 128
CONFIGS = {"64": (TINY["F"][0], 16), "64, windows": (TINY["V"][0], 16), "128": (dict(TINY["F"][0], head_dim=128, num_attention_heads=8), 32)}


@pytest.fixture
def calls(monkeypatch):
    """Steps of any size share.  Every call of the kernels that do is checked on the spot; the list has their largest groups and longest prefixes."""
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    monkeypatch.setattr(CudaOps, "SHARED_PART", {BF16: 0.0, F32: 0.0})
    inner, seen = CudaOps._shared_decode, []

    def checked(self, q, k_cache, v_cache, out, meta, H, KV, D, scale, size):
        inner(self, q, k_cache, v_cache, out, meta, H, KV, D, scale, size)
        alone = types.SimpleNamespace(decode_segs=meta.decode_segs, seg_q_start=meta.seg_q_start, seg_kv_len=meta.seg_kv_len, block_table=meta.block_table, table_rows=meta.table_rows,
                                      page_size=meta.page_size, shared_start=meta.decode_segs.new_zeros(1), shared_len=meta.decode_segs[:0])
        want, weight, reach = shared_prefix_attention64(q, k_cache.nan_to_num(0.0, 0.0, 0.0), v_cache.nan_to_num(0.0, 0.0, 0.0), alone, H, KV, D, scale)
        rows = meta.seg_q_start[meta.decode_segs.long()].long().cpu()
        o, w, a = out.cpu().double()[rows], want[rows], weight[rows]
        half, n = torch.finfo(q.dtype).eps / 2, int(meta.seg_kv_len.max())          # (as in test_shared_attention.check)
        per_weight = 2 * (D * 2.0 ** -24 * reach + 2.0 ** -22) + (n + 8) * 2.0 ** -24 + (half if q.dtype == BF16 else 0.0)
        assert ((o - w).abs() <= half * w.abs() + per_weight * a * (1 + half)).all()
        starts = meta.shared_start.tolist()
        assert meta.max_shared_rows >= max(b - a for a, b in zip(starts, starts[1:])) and meta.max_kv_len >= n
        shared = [s for s, a, b in zip(meta.shared_len.tolist(), starts, starts[1:]) if b - a > 1]
        assert meta.max_shared_len == max(shared, default=0)
        seen.append((meta.max_shared_rows, meta.max_shared_len, q.dtype))
    monkeypatch.setattr(CudaOps, "_shared_decode", checked)
    return seen


def model(tmp_path, name):
    cfg, page = CONFIGS[name]
    d = str(tmp_path / "model")
    write_random_model(cfg, d, seed=5, std=0.2, norm_init="uniform")
    return d, cfg, page


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_searches_in_float32(tmp_path, calls, name):
    d, cfg, page = model(tmp_path, name)
    llm = engine(d, page, "cuda:0")
    prompts = [random_tokens(cfg["vocab_size"], n, seed=n) for n in (5, page, 3 * page + 1)]
    check(llm, prompts, BeamParams(num_beams=4, max_new_tokens=2 * page + 3, ignore_eos=True), TOL)
    assert max(rows for rows, _, _ in calls) == 4 and max(n for _, n, _ in calls) >= 3 * page


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_calls_in_bfloat16(tmp_path, calls, name):
    """Beams that part and come together again, prompts that end before others, one after the other in waves."""
    d, cfg, page = model(tmp_path, name)
    llm = engine(d, page, "cuda:0", dtype="bfloat16", max_num_seqs=14, kv_cache_tokens=4096)
    prompts = [random_tokens(cfg["vocab_size"], n, seed=n) for n in (7 * page + 3, 5, 2 * page, 4 * page - 1)]
    free = llm.beam_search(prompts, BeamParams(num_beams=6, max_new_tokens=page + 5, ignore_eos=True))
    llm.eos_ids = {b.tokens[5] for beams in free for b in beams[:2]}
    llm.beam_search(prompts, BeamParams(num_beams=6, max_new_tokens=page + 5))
    llm.cache.check_invariants()
    assert max(rows for rows, _, _ in calls) == 6 and max(n for _, n, _ in calls) >= 7 * page and all(t is BF16 for _, _, t in calls)
