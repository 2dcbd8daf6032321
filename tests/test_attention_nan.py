"""Decoded tokens' attention where queries, keys or values that a row sees hold NaN: NaN exactly where the formula in 64 bits has it, numbers elsewhere, and zeros for
entries without keys."""
import math

import pytest
import torch

from mini_inference_b200.ops import CudaOps
from tests.ref_beam import shared_prefix_attention64
from tests.test_shared_attention import BF16, F32, problem

DEV = "cuda:0"
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from mini_inference_b200.ops import get_ops
    return get_ops(DEV)


def place_of(meta, r, j):
    """(page, place in it) of key j of row r."""
    e = int(meta.decode_segs[r])
    row = e if meta.table_rows is None else int(meta.table_rows[e])
    return int(meta.block_table[row, j // meta.page_size]), j % meta.page_size


def check_nan(q, k, v, meta, H, KV, D, scale, got):
    """Outputs are NaN where the formula's are.  The others are held to what clean inputs are held to: a row that sees no NaN has none in its sums."""
    want = shared_prefix_attention64(q, k, v, meta, H, KV, D, scale)[0]
    size, reach = shared_prefix_attention64(q.nan_to_num(0.0), k.nan_to_num(0.0), v.nan_to_num(0.0), meta, H, KV, D, scale)[1:]
    rows = meta.seg_q_start[meta.decode_segs.long()].long().cpu()
    o, w, a = got.cpu().double()[rows], want[rows], size[rows]
    assert torch.equal(o.isnan(), w.isnan()), ((o.isnan() != w.isnan()).view(len(rows), H, D).any(-1).nonzero()[:8].tolist(), int(w.isnan().sum()))
    # as test_shared_attention.check: the output's rounding, each weight's score and exponential (twice), sums over n keys, bfloat16 weights rounded once more
    half, n = torch.finfo(q.dtype).eps / 2, int(meta.seg_kv_len.max())
    per_weight = 2 * (D * 2.0 ** -24 * reach + 2.0 ** -22) + (n + 8) * 2.0 ** -24 + (half if q.dtype == BF16 else 0.0)
    ok = (o - w).abs() <= half * w.abs() + per_weight * a * (1 + half)
    assert (ok | w.isnan()).all()
    return want


def spoiled(groups, H, KV, D, ps, dtype, where, seed, alone=()):
    """Queries, caches and lists with NaN: where "query": the second row's query of the last head; "key", "value": of the second row, its last key; "all": every
    query; "first key": the one that the group's rows share."""
    q, k, v, meta = problem(groups, H, KV, D, ps, dtype, seed=seed, garbage=0.0, alone=alone)
    q = q.clone()
    tok = int(meta.seg_q_start[int(meta.decode_segs[1])])
    if where == "query":
        q[tok, H * D - 3] = math.nan
    elif where == "all":
        q.fill_(math.nan)
    else:
        page, at = place_of(meta, 1, 0 if where == "first key" else int(meta.seg_kv_len[int(meta.decode_segs[1])]) - 1)
        (v if where == "value" else k)[page, KV - 1, at, 5] = math.nan
    return q, k, v, meta


WHERE = ["query", "all", "key", "value", "first key"]
# one split and several; clusters, counters and a launch of its own for the merge
FORMS = [dict(), dict(force_splits=2), dict(force_splits=4), dict(force_splits=5, cluster_merge=False), dict(force_splits=6, fused_merge=False), dict(force_splits=12)]
LENS = [(0, [1, 2, 0, 40]), (0, [1500, 1400, 33, 0])]


@gpu
@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("H,KV,D,ps,dtype", [(8, 2, 128, 16, BF16), (6, 2, 64, 32, BF16), (6, 3, 48, 4, BF16), (6, 2, 64, 16, F32), (6, 3, 32, 4, F32), (8, 2, 128, 16, F32)])
def test_rows_one_by_one(ops, monkeypatch, H, KV, D, ps, dtype, form, where):
    """paged_attention's decoded tokens, on every kernel and merge that takes them."""
    for name, value in FORMS[form].items():
        monkeypatch.setattr(ops, name, value)
    for lens in LENS:
        q, k, v, meta = spoiled([lens], H, KV, D, ps, dtype, where, seed=D + form)
        meta.shared_start, meta.prefill_tiles, meta.tile = None, meta.decode_segs[:0].view(0, 2), 64
        got = ops.paged_attention(q, k, v, meta, H, KV, D, D ** -0.5, None)
        ops.check_errors()
        meta.shared_start = torch.zeros(1, dtype=torch.int32)
        meta.shared_len = meta.shared_start[:0]
        want = check_nan(q, k, v, meta, H, KV, D, D ** -0.5, got)
        assert want.isnan().any()


@gpu
@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("H,KV,D,ps,dtype", [(8, 2, 128, 16, BF16), (6, 2, 64, 32, BF16), (6, 3, 48, 4, BF16), (6, 2, 64, 16, F32), (8, 2, 128, 16, F32)])
def test_small_calls_of_the_operator(ops, H, KV, D, ps, dtype, where):
    """shared_prefix_attention where calls that read little go."""
    for groups in ([(0, [1, 2, 0, 40])], [(32, [33, 40, 32])], [(512, [1500, 1400, 512, 0])], [(64, [8100, 8200])]):
        q, k, v, meta = spoiled(groups, H, KV, D, ps, dtype, where, seed=D)
        got = ops.shared_prefix_attention(q, k, v, meta, H, KV, D, 0.1)
        ops.check_errors()
        check_nan(q, k, v, meta, H, KV, D, 0.1, got)


@gpu
@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("H,KV,D,ps,dtype", [(8, 2, 128, 16, BF16), (32, 8, 128, 16, BF16), (6, 2, 64, 32, BF16), (16, 1, 128, 64, BF16), (6, 2, 64, 16, F32), (8, 2, 128, 16, F32)])
def test_shared_prefixes(ops, monkeypatch, H, KV, D, ps, dtype, where):
    """On the kernels that share: prefixes and tails of one piece and of many, tails of a single key, rows alone."""
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    for groups in ([(64, [65, 65, 90])], [(0, [1, 1, 3])], [(2048, [2049, 2500, 2060, 2048]), (128, [129, 140])], [(512, [513] * 33), (64, [0, 70, 65])], [(4096, [4200, 6000])]):
        q, k, v, meta = spoiled(groups, H, KV, D, ps, dtype, where, seed=D, alone=(1, 300))
        assert ops._shared_bytes(q, k, v, meta, H, KV, D) > 0
        got = ops.shared_prefix_attention(q, k, v, meta, H, KV, D, 0.1)
        ops.check_errors()
        want = check_nan(q, k, v, meta, H, KV, D, 0.1, got)
        assert want.isnan().any()
