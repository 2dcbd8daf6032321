"""Decode attention over a shared prefix where rows end inside it: a group whose rows are all shorter than what they are said to share, some of them, and infinite
values that only the longer rows see.  Whatever lies behind a row's last key (in its pages, and in the pages that its table names behind them) may be anything."""
import math

import pytest
import torch

from tests.ref_beam import shared_prefix_attention64
from tests.test_shared_attention import BF16, F32, check, form, ops, problem      # noqa: F401  (fixtures: every test on the kernels by the rule and on those that share)

gpu = pytest.mark.gpu

SHAPES = [(8, 2, 128, 16, BF16), (6, 2, 64, 32, BF16), (16, 1, 128, 64, BF16), (6, 2, 128, 128, BF16), (8, 8, 64, 8, BF16), (8, 2, 128, 16, F32), (8, 8, 64, 16, F32), (10, 2, 128, 32, F32),
          (6, 3, 48, 4, BF16)]
GROUPS = {
    "all shorter": [(64, [10, 20])],
    "all shorter, beside others": [(320, [10, 300, 319]), (64, [65, 70]), (1000, [1, 999]), (77, [76, 76])],
    "some shorter": [(64, [10, 70, 65, 63]), (320, [400, 1, 320, 319, 0])],
    "one has them all": [(512, [100, 511, 700, 3])],
    "first ones empty and short": [(160, [0, 5, 161, 0, 170])],
    "many rows": [(208, [1 + 7 * i for i in range(60)]), (512, [511] * 33 + [600])],
    "long": [(4096, [4000, 4100, 2048, 4097]), (3000, [2999, 1500])],
}


def whole_pages(groups, ps):
    """Groups whose pages hold the same keys for all rows, whatever their first row's length: shared keys in whole pages where a row ends inside them."""
    return [(shared if min(lens) >= shared else shared // ps * ps, lens) for shared, lens in groups]


@gpu
@pytest.mark.parametrize("garbage", [math.nan, math.inf])
@pytest.mark.parametrize("H,KV,D,ps,dtype", SHAPES)
@pytest.mark.parametrize("name", GROUPS)
def test_rows_that_end_inside_the_prefix(ops, name, H, KV, D, ps, dtype, garbage):      # noqa: F811
    q, k, v, meta = problem(whole_pages(GROUPS[name], ps), H, KV, D, ps, dtype, seed=len(name) + D, garbage=garbage)
    check(ops, q, k, v, meta, H, KV, D)


@gpu
@pytest.mark.parametrize("H,KV,D,ps,dtype", [(8, 2, 128, 16, BF16), (6, 2, 64, 32, BF16), (8, 2, 128, 16, F32), (8, 8, 64, 16, F32)])
def test_infinite_values_that_only_longer_rows_see(ops, H, KV, D, ps, dtype):      # noqa: F811
    """A row that ends in front of them is as if they were not there; one that sees them has no finite number in their column."""
    lens = [400, 192, 320, 17, 0, 385]
    q, k, v, meta = problem([(384, lens)], H, KV, D, ps, dtype, seed=5, garbage=0.0)
    at = 350
    page = int(meta.block_table[0, at // ps])
    clean = v.clone()
    v[page, :, at % ps, 7], v[page, :, at % ps, 9] = math.inf, -math.inf
    got = ops.shared_prefix_attention(q, k, v, meta, H, KV, D, 0.1)
    ops.check_errors()
    want, size, reach = shared_prefix_attention64(q, k, clean, meta, H, KV, D, 0.1)
    half = torch.finfo(dtype).eps / 2
    per_weight = 2 * (D * 2.0 ** -24 * reach + 2.0 ** -22) + (max(lens) + 8) * 2.0 ** -24 + (half if dtype == BF16 else 0.0)      # (as in check)
    o = got.cpu().double().view(len(lens), H, D)
    near = ((got.cpu().double() - want).abs() <= half * want.abs() + per_weight * size * (1 + half)).view(len(lens), H, D)
    for r, n in enumerate(lens):
        sees = torch.zeros(D, dtype=torch.bool)
        sees[[7, 9]] = n > at
        assert near[r][:, ~sees].all() and not o[r][:, sees].isfinite().any(), r


# (rows of each group) of calls whose groups are very unlike
UNLIKE = [(64,) + (1,) * 256, (1000,) + (1,) * 1000, (1, 1, 300, 2, 1) + (3,) * 100]


@pytest.mark.parametrize("sizes", UNLIKE)
@pytest.mark.parametrize("H,KV,D", [(32, 8, 128), (4, 1, 64), (16, 16, 64)])
def test_scratch_goes_by_the_rows_and_not_by_the_largest_group(sizes, H, KV, D):
    """Prefix pieces take at most four copies of every row (one in float32), tails the same, and each of a few hundred blocks one piece more of 128 rows (32)."""
    from mini_inference_b200.ops import load_calls
    lib, R = load_calls(), sum(sizes)
    for entry, copies, tile in ((lib.mi_attn_shared_tc_bytes, 4, 128), (lib.mi_attn_shared_f32_bytes, 1, 32)):
        size = entry(R, len(sizes), max(sizes), H, KV, D, 16)
        blocks = 2 * 160
        assert 0 < size <= (2 * copies * R * H + 2 * blocks * tile) * (4 * D + 8) + 64 * R + 8192
        assert size <= 2 ** 31                                     # (the largest of these took 15.7 GB when every group had the room of the largest)


@gpu
@pytest.mark.parametrize("sizes", UNLIKE)
@pytest.mark.parametrize("H,KV,D,dtype", [(4, 1, 64, BF16), (8, 2, 128, BF16), (4, 1, 64, F32)])
def test_groups_unlike_one_another(ops, sizes, H, KV, D, dtype):      # noqa: F811
    groups = [(32 if n > 1 else 0, [33 + 5 * (i % 7) if i % 11 else 20 + i % 11 for i in range(n)]) for n in sizes]
    q, k, v, meta = problem(groups, H, KV, D, 16, dtype, seed=sum(sizes))
    check(ops, q, k, v, meta, H, KV, D)


@gpu
@pytest.mark.parametrize("H,KV,D,ps,dtype", [(128, 1, 128, 16, BF16), (96, 2, 64, 16, BF16), (40, 1, 128, 16, BF16), (33, 1, 64, 32, BF16), (65, 1, 64, 256, BF16), (64, 64, 64, 16, BF16), (34, 2, 128, 16, BF16),
                                             (32, 1, 64, 16, F32), (17, 1, 128, 8, F32), (21, 3, 64, 16, F32), (48, 48, 64, 1, F32)])
def test_many_query_heads_of_a_key_head(ops, H, KV, D, ps, dtype):      # noqa: F811
    """A row alone fills a tile, or half of one and a head more; many key heads."""
    for groups in ([(256, [257, 300, 256, 12])], [(0, [700]), (64, [65 + 3 * i for i in range(9)])]):
        q, k, v, meta = problem(groups, H, KV, D, ps, dtype, seed=H + KV)
        check(ops, q, k, v, meta, H, KV, D)
