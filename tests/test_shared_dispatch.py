"""Which decode steps go to the kernels that share prefixes: the rule on the host, and what a step of beams tells it."""
import types

import pytest
import torch

from mini_inference_b200.engine.batch import BatchBuilder, StepEntry, shared_of
from mini_inference_b200.cache import CacheManager
from mini_inference_b200.ops import CudaOps
from mini_inference_b200.parts.attention import paged_attention_step_arrays
from mini_inference_b200.parts.base import KVCacheNeed
from tests.ref_beam import BeamRefOps
from tests.test_beam_operators import bare

BF16, F32 = torch.bfloat16, torch.float32


def pays(dtype, rows, keys, shared, KV=8, D=128):
    q = torch.zeros(1, dtype=dtype)
    meta = types.SimpleNamespace(decode_segs=range(rows), max_kv_len=keys)
    if shared is not None:
        meta.max_shared_len = shared
    return bare()._sharing_pays(q, meta, KV, D, dtype is BF16)


def test_calls_that_read_little_are_read_row_by_row():
    # 16 rows of 2,048 keys over 8 heads of 128 are 128 MB to the byte
    assert not pays(BF16, 4, 560, 512) and not pays(BF16, 16, 2048, 2000) and pays(BF16, 16, 2049, 2000) and pays(BF16, 64, 4352, 4096)
    assert not pays(F32, 8, 4096, 4000) and pays(F32, 16, 4352, 4200) and not pays(F32, 13, 1604, 1504)


def test_float32_calls_that_share_little_are_read_row_by_row():
    for rows, keys, shared in ((64, 2048, 0), (64, 2048, 64), (64, 2304, 2048), (64, 9192, 8000), (16, 5120, 4096)):
        assert not pays(F32, rows, keys, shared)
        assert pays(F32, rows, keys, None)                         # nothing is said: by what is read alone
        assert pays(BF16, rows, keys, shared)
    for rows, keys, shared in ((64, 2064, 2048), (64, 2176, 2048), (16, 4352, 4096), (16, 32500, 32000), (8, 17000, 16000)):
        assert pays(F32, rows, keys, shared)


def builder(pages=200):
    cache = CacheManager([KVCacheNeed(2, 8)], 4, pages, 16, 80, dtype=torch.float32)
    return cache, BatchBuilder(cache, "cpu", {"paged_attention": paged_attention_step_arrays}, tile=64, vocab_size=10)


def family(cache, name, n, length, more):
    seq = cache.admit((name, 0))
    assert cache.ensure(seq, length)
    cache.commit(seq, length)
    seqs = [seq] + cache.fork(seq, [(name, i) for i in range(1, n)])
    cache.reorder([(seqs, [0] * n)], BeamRefOps())
    for s in seqs:
        assert cache.ensure(s, length + more + 1)
        cache.commit(s, length + more)
    return seqs


def test_what_a_step_of_beams_says():
    """Groups, their common keys and the largest of both: of one prompt, of several, of a beam alone beside others and with a prompt's portion between them."""
    cache, build = builder()
    a, b, c = family(cache, "a", 3, 21, 2), family(cache, "b", 2, 9, 4), family(cache, "c", 1, 33, 1)
    other, prompt = cache.admit("other"), cache.admit("prompt")
    for s, n in ((other, 12), (prompt, 5)):
        assert cache.ensure(s, 20)
        cache.commit(s, n)

    def step(*seqs, portion=()):
        entries = [StepEntry(s, [1] * (3 if s in portion else 1), [0]) for s in seqs]
        batch = build.build(entries)
        view = batch.group_view(0, "paged_attention")
        start, length = (None, None) if batch.extras["paged_attention"].get("shared_start") is None else (view.shared_start.tolist(), view.shared_len.tolist())
        return start, length, view.max_shared_rows, view.max_shared_len
    assert step(*a) == ([0, 3], [20], 3, 20)
    assert step(*a, *b, *c) == ([0, 3, 5, 6], [20, 8, 32], 3, 20)  # one row shares with nobody
    assert step(*c) == ([0, 1], [32], 1, 0)
    assert step(a[0], other, *b) == ([0, 1, 2, 4], [20, 0, 8], 2, 8)
    assert step(a[0], prompt, a[1], a[2], portion=(prompt,)) == ([0, 1, 3], [20, 20], 2, 20)
    assert step(other, prompt)[2:] == (0, 0) and step(other, prompt)[0] is None
    assert shared_of([other, prompt], [1, 1]) is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_paged_attention_with_a_scale_below_zero(monkeypatch, dtype):
    """paged_attention takes any scale; the kernels that share take the largest product for the largest score, which asks for a positive one."""
    from mini_inference_b200.ops import get_ops
    from tests.test_shared_attention import check, problem
    ops = get_ops("cuda:0")
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    q, k, v, meta = problem([(160, [161, 200, 300]), (64, [65, 90])], 8, 2, 128, 16, dtype, seed=4)
    q = (q.float() * 12).to(dtype)                                 # products of some hundred: their weights by the wrong end overflow
    meta.prefill_tiles, meta.tile = meta.decode_segs[:0].view(0, 2), 64
    got = ops.paged_attention(q, k, v, meta, 8, 2, 128, -1.0, None)
    check(ops, -q, k, v, meta, 8, 2, 128, scale=1.0, got=got)      # the same scores, exactly
    got = ops.paged_attention(q, k, v, meta, 8, 2, 128, 1.0, None)
    check(ops, q, k, v, meta, 8, 2, 128, scale=1.0, got=got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_token_in_a_row_of_any_width(monkeypatch, dtype):
    """A single token has no distance to the next one, whatever its stride says."""
    from mini_inference_b200.ops import get_ops
    from tests.test_shared_attention import check, problem
    ops = get_ops("cuda:0")
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    q, k, v, meta = problem([(0, [300])], 8, 2, 64, 16, dtype, seed=4)
    for width in (8 * 64 + 1, 8 * 64 + 3, 8 * 64 + 8):
        wide = torch.randn(1, width, device=q.device).to(dtype)
        check(ops, wide[:, :8 * 64], k, v, meta, 8, 2, 64)
    check(ops, wide.as_strided((1, 8 * 64), (0, 1)), k, v, meta, 8, 2, 64)
