"""Decode attention over a shared prefix (CudaOps.shared_prefix_attention) against a plain statement in 64 bits, and what it refuses."""
import math
import types

import pytest
import torch

from mini_inference_b200.ops import CudaOps
from tests.ref_beam import shared_prefix_attention64
from tests.test_beam_operators import bare, starts

DEV = "cuda:0"
gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from mini_inference_b200.ops import get_ops
    return get_ops(DEV)


def problem(groups, H, KV, D, ps, dtype, seed=0, alone=(), garbage=math.nan, extra_tokens=0, slots=False):
    """groups: (shared keys, [keys of each row, shared ones included]); alone: lengths of rows in no group.  Whatever no row may see (the null page, the unused
    ends of pages) holds `garbage`.  extra_tokens: tokens of a prompt entry in front of every row, so that rows are not neighbours."""
    g = torch.Generator().manual_seed(seed)
    lens = [n for _, ns in groups for n in ns] + list(alone)
    R = len(lens)
    pages = [[] for _ in range(R)]
    count = [1]

    def take():
        count[0] += 1
        return count[0] - 1
    r = 0
    copies = []                                                   # (page, page of the group's first row, keys) that hold the same keys
    for shared, ns in groups:
        full = [take() for _ in range(shared // ps)]
        for i, n in enumerate(ns):
            own = [take() for _ in range(-(-n // ps) - len(full))]
            pages[r + i] = full + own
            if i and shared % ps and own and pages[r][len(full):]:
                copies.append((own[0], pages[r][len(full)], shared % ps))
        r += len(ns)
    for i, n in enumerate(alone):
        pages[r + i] = [take() for _ in range(-(-n // ps))]
    perm = torch.randperm(count[0] - 1, generator=g) + 1
    at = lambda p: int(perm[p - 1])                               # noqa: E731
    k, v = (torch.randn(count[0], KV, ps, D, generator=g) for _ in range(2))
    for p, first, n in copies:
        k[at(p), :, :n], v[at(p), :, :n] = k[at(first), :, :n], v[at(first), :, :n]
    seen = torch.zeros(count[0], ps, dtype=torch.bool)
    for r, n in enumerate(lens):
        for j in range(n):
            seen[at(pages[r][j // ps]), j % ps] = True
    k.masked_fill_(~seen[:, None, :, None], garbage)
    v.masked_fill_(~seen[:, None, :, None], garbage)
    width = max([len(p) for p in pages] + [1])
    step = 2 if extra_tokens else 1                               # entries: (a prompt entry,) the row
    entries = R * step
    segs = [step * i + step - 1 for i in range(R)]
    q_start = [0]
    for e in range(entries):
        q_start.append(q_start[-1] + (extra_tokens if extra_tokens and e % 2 == 0 else 1))
    kv_len = [1] * entries
    order = torch.randperm(entries, generator=g).tolist() if slots else list(range(entries))
    table = torch.zeros(entries + 3, width, dtype=torch.int32)
    for r, e in enumerate(segs):
        kv_len[e] = lens[r]
        table[order[e], :len(pages[r])] = torch.tensor([at(p) for p in pages[r]], dtype=torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).to(DEV)    # noqa: E731
    meta = types.SimpleNamespace(decode_segs=i32(segs), seg_q_start=i32(q_start), seg_kv_len=i32(kv_len), block_table=table.to(DEV), max_pages=width, page_size=ps,
                                 table_rows=i32(order) if slots else None, max_kv_len=max(lens + [1]), shared_start=starts([len(ns) for _, ns in groups]).to(DEV),
                                 shared_len=i32([s for s, _ in groups]), max_shared_rows=max([len(ns) for _, ns in groups] + [0]))
    q = torch.randn(q_start[-1], (H + 2 * KV) * D, generator=g).to(dtype).to(DEV)[:, :H * D]
    return q, k.to(dtype).to(DEV), v.to(dtype).to(DEV), meta


@pytest.fixture(params=["by the rule", "shared at any size"], autouse=True)
def form(request, monkeypatch):
    """Calls that read little go to the kernels without sharing; every test runs on both."""
    if request.param != "by the rule":
        monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    return request.param


def check(ops, q, k, v, meta, H, KV, D, scale=None, got=None):
    scale = scale or D ** -0.5
    want, size, reach = shared_prefix_attention64(q, k.nan_to_num(0.0, 0.0, 0.0), v.nan_to_num(0.0, 0.0, 0.0), meta, H, KV, D, scale)
    if got is None:
        got = ops.shared_prefix_attention(q, k, v, meta, H, KV, D, scale)
        ops.check_errors()
    assert got.dtype == q.dtype and got.shape == want.shape
    rows = meta.seg_q_start[meta.decode_segs.long()].long().cpu()
    o, w, a = got.cpu().double()[rows], want[rows], size[rows]
    # the output is rounded once (half a step); a weight's score is a float32 sum of D products and its exponential is off by 2 units (weights and their sum: twice);
    # sums over n keys; bfloat16 runs round each weight once more (half a step)
    half = torch.finfo(q.dtype).eps / 2
    n = int(meta.seg_kv_len.max())
    per_weight = 2 * (D * 2.0 ** -24 * reach + 2.0 ** -22) + (n + 8) * 2.0 ** -24 + (half if q.dtype == BF16 else 0.0)
    bad = ~((o - w).abs() <= half * w.abs() + per_weight * a * (1 + half))
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist(), float((o - w).abs().nan_to_num(9.0).max()))


GROUPS = {
    "one beam": [(0, [1])],
    "four beams": [(64, [65, 70, 66, 80])],
    "short": [(16, [17, 18])],
    "prefix of one tile and a key": [(65, [66, 65, 90])],
    "several": [(160, [161, 200, 300]), (0, [5, 9]), (320, [321]), (32, [33, 34, 35, 36, 37, 38, 39])],
    "long": [(4096, [4097, 4300, 4099, 4600]), (1504, [1600, 1505])],
    "unaligned": [(77, [78, 100, 79]), (1003, [1004, 1100]), (7, [8, 9, 10])],
    "many rows": [(208, [209 + 3 * i for i in range(70)]), (512, [513] * 33)],
    "nothing behind the prefix": [(96, [96, 97, 96]), (128, [128, 128])],
    "no keys": [(64, [0, 70, 65]), (0, [0, 0]), (32, [40, 0])],
}
SHAPES = [(32, 8, 128, 16, BF16), (40, 8, 128, 16, BF16), (6, 2, 64, 32, BF16), (8, 8, 64, 8, BF16), (16, 1, 128, 64, BF16), (6, 2, 128, 128, BF16), (14, 2, 64, 16, BF16),
          (8, 2, 128, 16, F32), (8, 8, 64, 16, F32), (10, 2, 128, 32, F32), (6, 3, 32, 4, F32), (6, 3, 48, 4, BF16), (4, 2, 128, 24, BF16)]


@gpu
@pytest.mark.parametrize("H,KV,D,ps,dtype", SHAPES)
@pytest.mark.parametrize("name", GROUPS)
def test_shared_prefix_attention(ops, name, H, KV, D, ps, dtype, form):
    q, k, v, meta = problem(GROUPS[name], H, KV, D, ps, dtype, seed=len(name) + D)
    if (name == "no keys" and (ops._shared_bytes(q, k, v, meta, H, KV, D) <= 0 or form == "by the rule")):
        pytest.skip("the first row has no pages, so the others' own may hold other keys than the group's: the kernels that share")
    check(ops, q, k, v, meta, H, KV, D)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_in_no_group_between_prompts_in_slots(ops, dtype):
    q, k, v, meta = problem(GROUPS["several"], 8, 2, 128, 16, dtype, seed=3, alone=(1, 700, 64, 65), extra_tokens=3, slots=True)
    check(ops, q, k, v, meta, 8, 2, 128)
    meta.max_shared_rows = 3                                       # rows of a larger group than said are computed alone
    check(ops, q, k, v, meta, 8, 2, 128)
    meta.shared_start, meta.shared_len, meta.max_shared_rows = meta.shared_start[:1], meta.shared_len[:0], 0
    check(ops, q, k, v, meta, 8, 2, 128)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf, 3e38])
def test_what_no_row_sees_stays_out(ops, garbage, dtype):
    q, k, v, meta = problem(GROUPS["unaligned"] + GROUPS["four beams"], 8, 2, 64, 16, dtype, seed=5, garbage=garbage, alone=(33,))
    big = 3e38 if garbage == 3e38 else None
    clean = lambda t: torch.where(t.float().abs() > 1e38, torch.zeros_like(t), t) if big else t      # noqa: E731
    want_k, want_v = clean(k), clean(v)
    got = ops.shared_prefix_attention(q, k, v, meta, 8, 2, 64, 0.125)
    check(ops, q, want_k, want_v, meta, 8, 2, 64, got=got)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_far_apart(ops, dtype):
    """Maxima that grow from tile to tile, in the prefix and in the tail, and weights that vanish."""
    q, k, v, meta = problem([(640, [641, 900, 700]), (128, [1000, 129])], 8, 2, 128, 16, dtype, seed=6)
    for factor in (0.01, 8.0):
        check(ops, (q.float() * factor).to(dtype), k, v, meta, 8, 2, 128, scale=0.2)
    ramp = torch.linspace(0.1, 6.0, k.shape[0], device=DEV)[:, None, None, None]
    check(ops, q, (k.float() * ramp).to(dtype), v, meta, 8, 2, 128)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sharing_and_reading_alone_agree_in_the_engine_form(ops, dtype):
    """paged_attention with groups in its arrays and without: within what both are off."""
    q, k, v, meta = problem(GROUPS["several"], 32, 8, 128, 16, dtype, seed=8, garbage=0.0)
    meta.prefill_tiles, meta.tile = meta.decode_segs[:0].view(0, 2), 64
    got = ops.paged_attention(q, k, v, meta, 32, 8, 128, 128 ** -0.5, None)
    check(ops, q, k, v, meta, 32, 8, 128, got=got)
    meta.shared_start = None
    plain = ops.paged_attention(q, k, v, meta, 32, 8, 128, 128 ** -0.5, None)
    assert (got.float() - plain.float()).abs().max() <= (0.04 if dtype == BF16 else 1e-4)      # both within half a step and the weights' rounding of values below 5


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_streams_and_graphs(ops, dtype):
    H, KV, D = 16, 4, 128
    q, k, v, meta = problem(GROUPS["several"], H, KV, D, 16, dtype, seed=9)
    q = q.contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.shared_prefix_attention(q, k, v, meta, H, KV, D, 0.1)
    side.synchronize()
    check(ops, q, k, v, meta, H, KV, D, scale=0.1, got=got)
    graphs, outs, qs = [], [], [q.clone(), torch.randn_like(q.float()).to(dtype)]
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.shared_prefix_attention(qs[i], k, v, meta, H, KV, D, 0.1))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for turn in range(3):
        for x in qs:
            x.normal_()
        # lengths and groups that the graphs were not captured with
        meta.seg_kv_len.sub_((meta.seg_kv_len > 170 + turn).int())
        if turn == 1:
            meta.shared_len.sub_(16 * (meta.shared_len > 16).int())
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(qs, outs):
            check(ops, x, k, v, meta, H, KV, D, scale=0.1, got=out)
    ops.check_errors()


@gpu
def test_results_do_not_depend_on_the_call(ops):
    """The same call twice: the same bits."""
    q, k, v, meta = problem(GROUPS["long"], 32, 8, 128, 16, BF16, seed=10)
    a = ops.shared_prefix_attention(q, k, v, meta, 32, 8, 128, 0.1)
    for _ in range(5):
        assert torch.equal(a, ops.shared_prefix_attention(q, k, v, meta, 32, 8, 128, 0.1))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_beyond_32_bits(ops, dtype):
    """Pages whose offset passes 2^31 elements and, in bytes, 2^32."""
    H, KV, D, ps = 8, 2, 128, 16
    q, k, v, meta = problem([(320, [321, 400, 350])], H, KV, D, ps, dtype, seed=11)
    pages = (1 << 31) // (KV * ps * D) + 600
    big_k, big_v = (torch.zeros(pages, KV, ps, D, dtype=dtype, device=DEV) for _ in range(2))
    shift = pages - k.shape[0]
    big_k[shift:], big_v[shift:] = k, v
    want = ops.shared_prefix_attention(q, k, v, meta, H, KV, D, 0.1)
    meta.block_table = torch.where(meta.block_table > 0, meta.block_table + shift, meta.block_table).to(torch.int32)
    assert torch.equal(ops.shared_prefix_attention(q, big_k, big_v, meta, H, KV, D, 0.1), want)


@gpu
def test_as_many_entries_as_it_takes(ops):
    """1,900 rows in groups of four, and more than the kernel takes (computed row by row)."""
    for n in (475, 900):                                          # (zeros behind the keys where rows are computed alone; test_what_no_row_sees_stays_out has the other numbers)
        takes = 5 * n <= 4096
        q, k, v, meta = problem([(16, [17, 18, 19, 20])] * n, 4, 1, 64, 16, BF16, seed=12, garbage=math.nan if takes else 0.0)
        assert (ops._shared_bytes(q, k, v, meta, 4, 1, 64) > 0) == takes
        check(ops, q, k, v, meta, 4, 1, 64)


@gpu
@pytest.mark.parametrize("H,KV,D,ps,dtype", [(6, 3, 48, 4, BF16), (6, 3, 32, 4, F32), (10, 2, 128, 32, F32), (8, 2, 64, 16, F32), (32, 8, 128, 16, BF16), (6, 2, 64, 32, BF16)])
def test_entries_without_keys_computed_alone(ops, H, KV, D, ps, dtype, monkeypatch):
    """Zeros, in one piece and where the longest entry makes several, and nothing of what lies behind the keys."""
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 1 << 60, F32: 1 << 60})
    for groups in (GROUPS["no keys"], [(0, [0, 3000, 1]), (700, [700, 0, 701])]):
        q, k, v, meta = problem(groups, H, KV, D, ps, dtype, seed=13)
        check(ops, q, k, v, meta, H, KV, D)


@gpu
@pytest.mark.parametrize("H,KV,D,ps", [(16, 8, 128, 16), (8, 2, 64, 32)])
@pytest.mark.parametrize("lens", [[255, 257], [2048, 2047, 1], [4097, 4100], [8200], [300, 0, 8100], [1025] * 5, [513] * 17, [700] * 40])
def test_few_rows_of_all_lengths(ops, lens, H, KV, D, ps):
    """From one split to eight, blocks of either size, as clusters and without."""
    q, k, v, meta = problem([(min([n for n in lens if n]) // ps * ps, lens)], H, KV, D, ps, BF16, seed=len(lens))
    check(ops, q, k, v, meta, H, KV, D)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_query_rows_of_any_stride_and_more_rows_than_there_are(ops, dtype):
    H, KV, D = 8, 2, 128
    q, k, v, meta = problem(GROUPS["four beams"], H, KV, D, 16, dtype, seed=14)
    meta.max_shared_rows = 2 ** 31 - 1
    check(ops, q, k, v, meta, H, KV, D)
    check(ops, q[:1].expand(4, -1), k, v, meta, H, KV, D)          # all rows the same memory
    wide = torch.randn(4, H * D + 4, device=DEV).to(dtype)
    check(ops, wide[:, :H * D], k, v, meta, H, KV, D)              # rows that do not lie whole heads apart
    q, k, v, meta = problem(GROUPS["one beam"], H, KV, D, 16, dtype, seed=15)
    check(ops, torch.randn(3, H * D + 8, device=DEV).to(dtype)[1:2, 8:], k, v, meta, H, KV, D)
    check(ops, q.contiguous().as_strided((1, H * D), (0, 1)), k, v, meta, H, KV, D)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_caches_off_16_bytes_are_refused(ops, dtype):
    q, k, v, meta = problem(GROUPS["short"], 8, 2, 128, 16, dtype, seed=16)
    off = torch.zeros(k.numel() + 1, dtype=dtype, device=DEV)[1:].view(k.shape)
    for caches in ((off, v), (k, off)):
        with pytest.raises(ValueError, match="16 bytes"):
            ops.shared_prefix_attention(q, *caches, meta, 8, 2, 128, 0.1)


def test_refusals():
    me = bare()
    q, k = torch.zeros(4, 8 * 64), torch.zeros(3, 2, 16, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)           # noqa: E731
    meta = lambda **kw: types.SimpleNamespace(**{**dict(decode_segs=i32(0, 1, 2, 3), seg_q_start=i32(0, 1, 2, 3, 4), seg_kv_len=i32(5, 5, 5, 5), table_rows=None,      # noqa: E731
                                                        block_table=torch.zeros(4, 2, dtype=torch.int32), max_pages=2, page_size=16, max_kv_len=5,
                                                        shared_start=i32(0, 4), shared_len=i32(4), max_shared_rows=4), **kw})
    good = (q, k, k, meta(), 8, 2, 64, 0.1)
    with pytest.raises(ValueError, match="cuda:0"):                # nothing wrong but the device
        me.shared_prefix_attention(*good)
    for change, error in (({0: q[:, :64]}, ValueError), ({0: q.bfloat16()}, TypeError), ({0: q.double(), 1: k.double(), 2: k.double()}, TypeError), ({1: k[:, :1]}, ValueError),
                          ({2: k.bfloat16()}, TypeError), ({1: k.transpose(0, 1).contiguous().transpose(0, 1)}, ValueError), ({4: 7}, ValueError), ({5: 3}, ValueError),
                          ({7: 0.0}, ValueError), ({7: math.nan}, ValueError), ({3: meta(page_size=8)}, ValueError), ({3: meta(shared_len=i32(4, 4))}, ValueError),
                          ({3: meta(shared_start=torch.tensor([0, 4]))}, TypeError), ({3: meta(seg_kv_len=torch.zeros(4))}, TypeError), ({3: meta(max_pages=3)}, ValueError),
                          ({3: meta(decode_segs=torch.zeros(4, 1, dtype=torch.int32))}, ValueError), ({0: torch.zeros(8 * 64, 4).t()}, ValueError)):
        args = list(good)
        for i, value in change.items():
            args[i] = value
        with pytest.raises(error):
            me.shared_prefix_attention(*args)
