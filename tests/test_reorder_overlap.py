"""reorder_rows refuses tensors that share memory, and takes those that only reach into one another: on the CPU, where the device is what is refused last."""
import random

import pytest
import torch

from tests.test_beam_operators import DEV, bare, check_reorder, gpu, make, random_groups, starts


def refused(tensors, dim=0):
    me, rows, start = bare(), torch.arange(2, dtype=torch.int32), starts((2,))
    with pytest.raises(ValueError, match="same memory|cuda:0") as e:
        me.reorder_rows(tensors, rows, rows, start, 2, dim=dim)
    return "same memory" in str(e.value)


def test_views_that_overlap():
    t = torch.zeros(8, 40)
    flat = t.view(-1)
    assert refused([t[:5], t[4:]])
    assert refused([t[:, :21], t[:, 20:]])
    assert refused([flat[:81].view(27, 3), flat[80:].view(-1, 4)])
    assert refused([t, t[3:4, 7:9]])
    assert refused([t[:, 5:9], t[6:7, 8:12]])
    assert refused([torch.zeros(3, 2), t[1:], t[:, 39:]])
    assert refused([t[:, :9], t.view(torch.int32)[2:5, 8:30]])
    assert refused([t.view(2, 4, 40), t[7:].view(1, 1, 40)], dim=1)


def test_views_that_lie_side_by_side():
    t = torch.zeros(8, 40)
    assert not refused([t[:4], t[4:]])
    assert not refused([t[:, :20], t[:, 20:]])
    assert not refused([t[:, 30:], t[:, :10], t[:, 10:30]])
    assert not refused([t[:, :10], t[3:4, 10:12], t[2:3, 38:]])
    assert not refused([t[1:, :10], t[:7, 30:]])
    assert not refused([t[2:2], t, torch.zeros(0, 3)])
    assert not refused([t[:, :0], t])
    assert not refused([t[:1, :3], t[1:]])


def test_against_every_byte():
    """Views of one buffer at random: what shares a byte is refused, and what does not is taken where the rows' distances are the same (or one is in one piece)."""
    rng = random.Random(3)
    counts = [0, 0]
    for _ in range(3000):
        width = rng.randint(1, 12)
        base, views, seen = torch.zeros(80, dtype=torch.uint8), [], []
        for _ in range(2):
            w = width if rng.random() < 0.7 else rng.randint(1, 12)
            row, n, at = rng.randint(1, w), rng.randint(1, 5), rng.randint(0, 12)
            v = base.as_strided((n, row), (w, 1), at)
            views.append((v, w if n > 1 and row < w else 0))
            seen.append({at + i * w + j for i in range(n) for j in range(row)})
        same = refused([v for v, _ in views])
        if seen[0] & seen[1]:
            assert same
        elif 0 in (views[0][1], views[1][1]) or views[0][1] == views[1][1]:
            assert not same
        counts[same] += 1
    assert min(counts) > 300


@gpu
def test_columns_of_wider_slots():
    """Several states as columns of one wider tensor."""
    from mini_inference_b200.ops import get_ops
    ops = get_ops(DEV)
    rows, parents, start = random_groups((6, 6), 20, seed=7)
    wide = make((20, 700), torch.float32, 8)
    check_reorder(ops, [wide[:, :128], wide[:, 640:], wide[:, 129:640]], rows, parents, start, 6)
    with pytest.raises(ValueError, match="same memory"):
        ops.reorder_rows([wide[:, :128], wide[:, 127:]], rows.to(DEV), parents.to(DEV), start.to(DEV), 6)
