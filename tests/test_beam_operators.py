"""Beam search's operators alone: beam_select and reorder_rows against plain statements in 64 bits (tests/ref_beam.py), and what they refuse."""
import math

import pytest
import torch

from mini_inference_b200.ops import CudaOps
from tests.ref_beam import beam_select64, reorder_rows_plain

DEV = "cuda:0"
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from mini_inference_b200.ops import get_ops
    return get_ops(DEV)


def starts(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def check_select(ops, logits, scores, sizes, num):
    start = starts(sizes)
    want, rows, tokens = beam_select64(logits, scores, start, num)
    got = ops.beam_select(logits.to(DEV) if logits.device.type == "cpu" else logits, scores.to(DEV), start.to(DEV), num)
    assert [t.dtype for t in got] == [torch.float32, torch.int32, torch.int32] and all(t.shape == (len(sizes), num) for t in got)
    assert torch.equal(got[1].cpu(), rows) and torch.equal(got[2].cpu(), tokens)
    v = got[0].cpu().double()
    live = rows >= 0
    assert torch.equal(v == -math.inf, ~live)
    # the value itself is rounded once to float32 (half a step: 2^-24 of it); sums of exponentials are kept to 1e-9 and their logarithm adds that
    assert ((v - want)[live].abs() <= want[live].abs() * 2.0 ** -24 + 1e-8).all()


def model_logits(R, V, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * std
    x[torch.arange(R)[:, None], torch.randint(0, V, (R, 6), generator=g)] += torch.rand(R, 6, generator=g) * 10
    return x, -torch.rand(R, generator=g) * 30


@gpu
@pytest.mark.parametrize("sizes,V,num", [
    ((1,), 1, 1), ((1,), 5, 8), ((3, 1), 7, 128), ((4,), 255, 8), ((4,), 2048, 8), ((2, 5), 2049, 10), ((2, 5), 2047, 128), ((1, 2, 3), 4097, 3),
    ((8,), 8193, 16), ((5,), 50257, 10), ((4, 4), 151936, 8), ((32,), 32768, 64), ((1, 40, 3), 999, 33), ((8,) * 40, 16411, 16), ((100,), 1200, 128), ((300,), 77, 5),
])
def test_beam_select(ops, sizes, V, num):
    x, s = model_logits(sum(sizes), V, seed=V + num)
    check_select(ops, x, s, sizes, num)


@gpu
def test_beam_select_ties_go_to_the_lower_row_and_token(ops):
    x, _ = model_logits(1, 3000, seed=1)
    x = x.round().repeat(4, 1)                                   # many equal logits, four equal beams
    check_select(ops, x, torch.full((4,), -3.0), (4,), 24)
    check_select(ops, torch.zeros(3, 20001), torch.tensor([-1.0, -0.5, -0.5]), (3,), 128)          # every token ties: more than fit
    check_select(ops, torch.zeros(70, 5000), torch.full((70,), -2.0), (70,), 128)
    x = torch.zeros(2, 9000)
    x[0, ::2], x[1, 1::3] = -0.0, 1.0                            # -0 is 0
    check_select(ops, x, torch.zeros(2), (1, 1), 40)
    x = torch.zeros(1, 4000)
    x[0, 100:200] = 1e-30                                        # larger logits come first even where their values round to the same
    check_select(ops, x, torch.zeros(1), (1,), 128)


@gpu
def test_beam_select_rows_that_offer_nothing(ops):
    x, s = model_logits(9, 5000, seed=3)
    x[0] = -math.inf                                             # nothing allowed
    x[1, 4000] = math.nan
    x[2, 17] = math.inf
    s[3], s[4], s[5] = -math.inf, math.nan, math.inf
    x[6, :4990] = -math.inf                                      # ten tokens left
    x[7, 2048:] = -math.inf
    x[7, :2048] = torch.finfo(torch.float32).min                 # the type's lowest value is a score like another
    for sizes in ((9,), (3, 3, 3), (7, 0, 2), (6, 1, 1, 1), (0, 9, 0)):
        check_select(ops, x, s, sizes, 24)
    check_select(ops, x[:3], s[:3], (3,), 5)


@gpu
def test_beam_select_wide_range(ops):
    """Logits far apart, and a maximum far from zero, either side."""
    for shift, scale in ((0.0, 60.0), (3e4, 5.0), (-3e4, 5.0), (1e30, 0.0), (0.0, 1e-3)):
        x, s = model_logits(6, 12345, seed=9)
        check_select(ops, x * scale + shift, s, (2, 4), 20)


@gpu
def test_beam_select_along_long_rows(ops):
    """So many rows that a block streams several tiles: logits that rise or fall along them, past a thousand and back, begin with nothing, or are all the same."""
    R, V = 300, 20003
    x, s = model_logits(R, V, seed=21)
    along = torch.linspace(0, 1, V)
    x[0:20] += along * 30
    x[20:40] -= along * 60
    x[40:60] += along * 3000 - 1500                              # below a thousand, then above
    x[60:80] -= along * 3000 - 1500
    x[80:100, :9001] = -math.inf
    x[100:120, 9001:] = -math.inf
    x[120:140] = 0.5
    x[140:150, ::2] = -math.inf
    x[150, 19000], x[151, 2] = math.nan, math.inf
    x[152:160] = x[152:160].round()
    x[160:170] += (torch.arange(V) % 8192 // 4096) * 2000        # up and down by turns
    check_select(ops, x, s, (100, 20, 20, 30, 130), 24)
    check_select(ops, x, s, (150, 150), 128)


@gpu
def test_beam_select_strides_streams_and_graphs(ops):
    x, s = model_logits(6, 10007, seed=4)
    wide = torch.full((6, 10050), math.nan, device=DEV)
    for off in (0, 1, 3, 4):                                     # rows that start on 4, 8 and 16 bytes
        view = wide[:, off:off + 10007]
        view.copy_(x)
        check_select(ops, view, s, (2, 4), 12)
    start, xd, sd = starts((2, 4)).to(DEV), x.to(DEV), s.to(DEV)
    want = ops.beam_select(xd, sd, start, 12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(xd, sd, start, 12)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):                                           # two graphs of the same call, replayed at the same time
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.beam_select(xd, sd, start, 12))
        graphs.append(graph)
    x2, s2 = model_logits(6, 10007, seed=5)
    xd.copy_(x2)
    sd.copy_(s2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    want = ops.beam_select(xd, sd, start, 12)
    assert all(torch.equal(a, b) for out in outs for a, b in zip(want, out))


@gpu
def test_beam_select_without_rows(ops):
    got = ops.beam_select(torch.empty(0, 100, device=DEV), torch.empty(0, device=DEV), starts((0, 0)).to(DEV), 3)
    assert (got[0] == -math.inf).all() and (got[1] == -1).all() and (got[2] == -1).all()
    got = ops.beam_select(torch.empty(2, 100, device=DEV), torch.empty(2, device=DEV), starts(()).to(DEV), 3)
    assert got[0].shape == (0, 3)


# ---------------------------------------------------------------- reorder_rows
def random_groups(sizes, N, seed):
    g = torch.Generator().manual_seed(seed)
    start = starts(sizes)
    rows = torch.randperm(N, generator=g)[:sum(sizes)].to(torch.int32)
    parents = torch.cat([torch.randint(0, n, (n,), generator=g) + a for a, n in zip(start.tolist(), sizes)] or [torch.empty(0)]).to(torch.int32)
    return rows, parents, start


def check_reorder(ops, tensors, rows, parents, start, most, dim=0):
    want = [t.detach().cpu().clone() for t in tensors]
    reorder_rows_plain(want, rows, parents, start, dim)
    ops.reorder_rows(tensors, rows.to(DEV), parents.to(DEV), start.to(DEV), most, dim=dim)
    for a, b in zip(tensors, want):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


def make(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, 256, (*shape[:-1], shape[-1] * torch.empty((), dtype=dtype).element_size()), generator=g, dtype=torch.uint8)       # any bits, NaN among them
    return t.to(DEV).view(dtype)


@gpu
@pytest.mark.parametrize("sizes", [(1,), (4,), (2, 7, 1, 16), (100,), (33, 64), (3,) * 50])
def test_reorder_rows(ops, sizes):
    rows, parents, start = random_groups(sizes, sum(sizes) + 9, seed=sum(sizes))
    N = sum(sizes) + 9
    tensors = [make((N, 16, 24), torch.float32, 1), make((N, 5), torch.int32, 2), make((N, 1027), torch.bfloat16, 3), make((N, 4096), torch.bfloat16, 4),
               make((N, 3), torch.uint8, 5), make((N, 1), torch.int64, 6), make((N, 2049), torch.float32, 7), make((N,), torch.float32, 8)]
    check_reorder(ops, tensors, rows, parents, start, max(sizes))


@gpu
def test_reorder_rows_cycles_and_many_tensors(ops):
    rows = torch.tensor([5, 2, 9, 1, 0, 7], dtype=torch.int32)
    for parents in ([1, 2, 3, 4, 5, 0], [1, 0, 3, 2, 5, 4], [0, 0, 0, 0, 0, 0], [5, 4, 3, 2, 1, 0], [0, 1, 2, 3, 4, 5], [3, 3, 0, 2, 2, 1]):
        tensors = [make((11, 8 + i), torch.float32, i) for i in range(70)]
        check_reorder(ops, tensors, rows, torch.tensor(parents, dtype=torch.int32), starts((6,)), 6)


@gpu
def test_reorder_pages_of_all_layers(ops):
    rows, parents, start = random_groups((8, 3), 40, seed=6)
    t = make((5, 2, 41, 2, 16, 64), torch.bfloat16, 3)
    check_reorder(ops, [t], rows + 1, parents, start, 8, dim=2)


@gpu
def test_reorder_rows_of_strided_slots(ops):
    """States as a view of wider slots, and rows that do not start on 16 bytes."""
    rows, parents, start = random_groups((6, 6), 20, seed=7)
    for cols, off in ((512, 0), (512, 1), (100, 3), (7, 2)):
        wide = make((20, 700), torch.float32, 8)
        check_reorder(ops, [wide[:, off:off + cols]], rows, parents, start, 6)


@gpu
def test_reorder_rows_leaves_what_points_outside(ops):
    start = starts((3, 3))
    rows, parents = torch.tensor([0, 99, 2, 3, -1, 5], dtype=torch.int32), torch.tensor([1, 0, 4, 5, 3, 4], dtype=torch.int32)
    check_reorder(ops, [make((7, 300), torch.float32, 1), make((3, 300), torch.float32, 2)], rows, parents, start, 3)
    check_reorder(ops, [make((7, 300), torch.float32, 1)], rows[:0], parents[:0], starts((0, 0)), 0)


@gpu
def test_reorder_rows_beyond_32_bits(ops):
    """Rows whose offset passes 4 GB."""
    t = torch.zeros(700001, 4096, dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([3, 699999, 350001], dtype=torch.int32, device=DEV)
    t[rows.long()] = make((3, 4096), torch.bfloat16, 9).nan_to_num()
    want = t[rows.long()][[1, 2, 0]]
    ops.reorder_rows([t], rows, torch.tensor([1, 2, 0], dtype=torch.int32, device=DEV), starts((3,)).to(DEV), 3)
    assert torch.equal(t[rows.long()], want)


@gpu
def test_reorder_rows_in_a_graph(ops):
    rows, parents, start = (v.to(DEV) for v in random_groups((8,), 12, seed=3))
    t = make((12, 3000), torch.float32, 1).nan_to_num()
    want = t.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reorder_rows([t], rows, parents, start, 8)
    for turn in range(3):
        parents.copy_(random_groups((8,), 12, seed=turn)[1])
        reorder_rows_plain([want], rows, parents, start)
        graph.replay()
        assert torch.equal(t, want)


# ---------------------------------------------------------------- refusals, on the CPU: the device is looked at last
def bare():
    me = CudaOps.__new__(CudaOps)
    me._device_index, me.launches = 0, 0
    return me


def test_beam_select_refuses():
    me, x, s, start = bare(), torch.zeros(4, 10), torch.zeros(4), starts((4,))
    for args, error in (((x.double(), s, start, 2), TypeError), ((x.bfloat16(), s, start, 2), TypeError), ((x, s.double(), start, 2), TypeError),
                        ((x, s, start.long(), 2), TypeError), ((x, s[:3], start, 2), ValueError), ((x[0], s, start, 2), ValueError),
                        ((x, s, start[:0], 2), ValueError), ((x, s, start, 0), ValueError), ((x, s, start, 129), ValueError), ((x[:, :0], s, start, 2), ValueError),
                        ((x.t().contiguous().t(), s, start, 2), ValueError), ((x[:1].expand(4, 10), s, start, 2), ValueError),
                        ((x, torch.zeros(8)[::2], start, 2), ValueError), ((x, s, start, 2), ValueError)):
        with pytest.raises(error, match="beam_select"):
            me.beam_select(*args)


def test_reorder_rows_refuses():
    me, t, rows, start = bare(), torch.zeros(6, 3, 4), torch.arange(4, dtype=torch.int32), starts((4,))
    for args, kw, error in ((([t], rows.long(), rows, start, 4), {}, TypeError), (([t], rows, rows[:3], start, 4), {}, ValueError),
                            (([t], rows, rows, start, 101), {}, ValueError), (([t], rows, rows, start, -1), {}, ValueError), (([t], rows, rows, start[:0], 4), {}, ValueError),
                            (([t], rows, rows, start, 4), dict(dim=3), ValueError), (([t], rows, rows, start, 4), dict(dim=-1), ValueError),
                            (([t.transpose(1, 2)], rows, rows, start, 4), {}, ValueError), (([t[:1].expand(6, 3, 4)], rows, rows, start, 4), {}, ValueError),
                            (([t[:, ::2]], rows, rows, start, 4), dict(dim=1), ValueError), (([t], rows, rows, start, 4), {}, ValueError)):
        with pytest.raises(error, match="reorder_rows"):
            me.reorder_rows(*args, **kw)


def test_reorder_rows_refuses_a_tensor_twice():
    me, t, rows, start = bare(), torch.zeros(6, 3, 4), torch.arange(4, dtype=torch.int32), starts((4,))
    for tensors in ([t, t], [t, torch.zeros(6, 1), t.view(6, 12)]):
        with pytest.raises(ValueError, match="same memory"):
            me.reorder_rows(tensors, rows, rows, start, 4)
    with pytest.raises(ValueError, match="cuda:0"):               # empty ones have no memory
        me.reorder_rows([t, torch.zeros(0, 3), torch.zeros(0, 5)], rows, rows, start, 4)


def test_reorder_plain_statement():
    """Every row gets what its parent held before the call, whatever the order."""
    t = torch.arange(6.0).view(6, 1)
    reorder_rows_plain([t], torch.tensor([0, 2, 4]), torch.tensor([1, 2, 0]), torch.tensor([0, 3]))
    assert t.flatten().tolist() == [2, 1, 4, 3, 0, 5]
