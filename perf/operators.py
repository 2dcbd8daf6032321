"""Operators of beam search as cases that can be timed and checked.

A case is one pass through an operator of the kernel namespace (mini_inference_b200.ops): where `own` is true the call that a user
makes of it, else its plain form in elementary torch operations.

kind      operator                  what it stands for in use
select    beam_select               a step's candidates: log-probabilities of every beam of a prompt over the vocabulary, the best
                                    `num` of all its beams (twice the beams, so that enough go on when some end)
reorder   reorder_rows              survivors take over their parents' last pages, or recurrent states, in place
attention shared_prefix_attention   a decode step's attention: beams (or samples) of a prompt share its pages and have tails of their own

Sizes are those of Qwen3 configurations (4B and 8B: 32 query heads over 8 key heads of 128, 36 layers; 14B: 40 over 8), of the
designs with matrix states (16 heads of 128 x 128), and generic odd ones.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False
DEV = "cuda:0"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one user, four beams, a short prompt: the call's fixed cost
        dict(name="attention_4_beams_512", kind="attention", rows="4", prefix="512", tail=48, heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # eight prompts of about 4,096 tokens, eight beams each
        dict(name="attention_8x8_beams_4096", kind="attention", rows="8,8,8,8,8,8,8,8", prefix="4096,4096,3904,4048,4096,2512,4096,3600", tail=256,
             heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # 64 samples of one long prompt
        dict(name="attention_64_samples_8192", kind="attention", rows="64", prefix="8192", tail=1000, heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # a document of 32,000 tokens, 16 beams, five query heads to a key head
        dict(name="attention_16_beams_32000", kind="attention", rows="16", prefix="32000", tail=500, heads=40, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # ragged groups, one of a single row and one without a prefix, small heads, pages of 32
        dict(name="attention_ragged_dim64", kind="attention", rows="5,1,9,3,2", prefix="1056,2016,480,0,32", tail=200, heads=24, kv_heads=4, dim=64, page=32,
             dtype="bfloat16"),
        # a float32 run
        dict(name="attention_float32", kind="attention", rows="5,8", prefix="1504,976", tail=100, heads=32, kv_heads=8, dim=128, page=16, dtype="float32"),
        # one user, four beams
        dict(name="select_4_beams_32768", kind="select", rows="4", vocab=32768, num=8, banned=0),
        # eight prompts of eight beams over Qwen3's vocabulary
        dict(name="select_8x8_beams_151936", kind="select", rows="8,8,8,8,8,8,8,8", vocab=151936, num=16, banned=0),
        # ragged groups (a prompt's first step has one row), an odd vocabulary, tokens that may not be chosen
        dict(name="select_ragged_100003", kind="select", rows="1,5,3,16,2", vocab=100003, num=32, banned=500),
        # four beams' last pages: 36 layers, keys and values
        dict(name="reorder_pages_4_beams", kind="reorder", form="pages", layers=36, row=16384, groups=1, beams=4, moved=3, sources=2),
        # eight prompts of eight beams
        dict(name="reorder_pages_8x8_beams", kind="reorder", form="pages", layers=36, row=16384, groups=8, beams=8, moved=6, sources=3),
        # recurrent layers: matrix states in float32, a convolution's last inputs in bfloat16, small integer states
        dict(name="reorder_states_8x4_beams", kind="reorder", form="states", layers=8, row=16 * 128 * 128, groups=8, beams=4, moved=3, sources=2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_groups(rng, most_groups, most_rows, total):
    out = [_log_int(rng, 1, most_rows) for _ in range(_log_int(rng, 1, most_groups))]
    while len(out) > 1 and sum(out) > total:
        out.pop()
    return out


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "select", "select", "reorder"])
    most = {m: max(work(c)[m] for c in listed() if c["kind"] == kind) for m in ("bytes", "flops")}
    while True:
        if kind == "attention":
            rows = _draw_groups(rng, 12, 64, 160)
            page = rng.choice([16, 16, 32])
            longest = _log_int(rng, 64, 24000)
            prefix = [rng.choice([longest, rng.randint(0, longest)]) // page * page for _ in rows]
            heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (40, 8, 128), (16, 8, 128), (24, 4, 64), (6, 2, 64), (8, 8, 64)])
            case = dict(kind=kind, rows=",".join(map(str, rows)), prefix=",".join(map(str, prefix)), tail=_log_int(rng, 1, 700), heads=heads, kv_heads=kv,
                        dim=dim, page=page, dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]))
            if case["dtype"] == "float32" and work(case)["flops"] > 4 * max(work(c)["flops"] for c in listed() if c.get("dtype") == "float32"):
                continue
        elif kind == "select":
            rows = _draw_groups(rng, 12, 32, 64)
            case = dict(kind=kind, rows=",".join(map(str, rows)), vocab=_log_int(rng, 300, 152000), num=_log_int(rng, 1, 64), banned=rng.choice([0, 7, 200]))
        else:
            beams = rng.randint(2, 32)
            sources = rng.randint(1, beams // 2)
            form = rng.choice(["pages", "states"])
            row = rng.choice([16384, 4096, 1024 * rng.randint(1, 40)]) if form == "pages" else _log_int(rng, 500, 400000)
            case = dict(kind=kind, form=form, layers=rng.randint(1, 48), row=row, groups=_log_int(rng, 1, 16), beams=beams,
                        moved=rng.randint(sources, beams if sources > 1 else beams - 1), sources=sources)
        w = work(case)
        if all(w[m] <= most[m] for m in w):
            return case


def _ints(text):
    return [int(v) for v in str(text).split(",")]


def _tails(case):
    """Keys that each row has of its own: 1 .. tail, spread."""
    n = sum(_ints(case["rows"]))
    return [1 + (i * 7919 + 5 * case["tail"]) % case["tail"] for i in range(n)]


# ---------------------------------------------------------------- inputs, from the seed alone
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 29)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(rows):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return out


def _members(rows):
    """[groups, most rows]: each group's rows, the absent ones -1; and where row r stands in that table."""
    most, start = max(rows), _starts(rows)
    table = [[start[g] + i if i < n else -1 for i in range(most)] for g, n in enumerate(rows)]
    place = [g * most + i for g, n in enumerate(rows) for i in range(n)]
    return torch.tensor(table, device=DEV), torch.tensor(place, device=DEV)


def _prepare_select(case, seed):
    g, rows, V = _generator(seed), _ints(case["rows"]), case["vocab"]
    R = sum(rows)
    # a language model's scores: a broad bulk and a few tokens far above it
    x = torch.empty(R, V, device=DEV).normal_(0.0, 2.0, generator=g)
    high = torch.randint(0, V, (R, 12), generator=g, device=DEV)
    x.scatter_add_(1, high, torch.empty(R, 12, device=DEV).uniform_(2.0, 12.0, generator=g))
    if case["banned"]:
        x[:, torch.randint(0, V, (case["banned"],), generator=g, device=DEV)] = -math.inf
    # running sums of log-probabilities, the best beam first
    s = -torch.empty(R, device=DEV).exponential_(0.4, generator=g)
    start = _starts(rows)
    for a, b in zip(start, start[1:]):
        s[a:b] = s[a:b].cumsum(0) - 20.0
    members, _ = _members(rows)
    return SimpleNamespace(kind="select", logits=x, scores=s, group_start=_i32(start), num=case["num"], members=members)


def _prepare_reorder(case, seed):
    g, L, row, G, B = _generator(seed), case["layers"], case["row"], case["groups"], case["beams"]
    n = G * B
    if case["form"] == "pages":                       # [layers, keys and values, pages, row]; the pages of others around them
        tensors, dim, N = [torch.empty(L, 2, 2 * n + 1, row, device=DEV, dtype=torch.bfloat16).normal_(0.0, 1.0, generator=g)], 2, 2 * n + 1
    else:                                             # [slots, row] a layer
        N, dim, tensors = n + 3, 0, []
        for i in range(L):
            tensors.append(torch.empty(N, row, device=DEV).normal_(0.0, 0.3, generator=g))
            tensors.append(torch.empty(N, 3 * 301 * (1 + i % 3), device=DEV, dtype=torch.bfloat16).normal_(0.0, 0.9, generator=g))
            tensors.append(torch.randint(0, 1000, (N, 1 + i % 3), generator=g, device=DEV, dtype=torch.int32))
    rows = (torch.randperm(N - 1, generator=g, device=DEV)[:n] + 1).to(torch.int32)
    parents = torch.arange(n, device=DEV).view(G, B)
    pick = torch.rand(G, B, generator=g, device=DEV).argsort(1)                  # per group: the first `sources` of these are the parents
    child = torch.arange(B, device=DEV)
    for k in range(G):                                # `moved` rows with another parent: first those that are no source, then sources that become another source's child
        order = pick[k].flip(0)[:case["moved"]]
        source = pick[k][:case["sources"]]
        take = source[child[:case["moved"]] % case["sources"]]
        same = take == order
        take = torch.where(same, source[(child[:case["moved"]] + 1) % case["sources"]], take)
        parents[k, order] = k * B + take
    return SimpleNamespace(kind="reorder", tensors=tensors, rows=rows, parents=parents.reshape(-1).to(torch.int32), group_start=_i32([k * B for k in range(G + 1)]),
                           beams=B, dim=dim)


def _prepare_attention(case, seed):
    g, rows, prefix, tails = _generator(seed), _ints(case["rows"]), _ints(case["prefix"]), _tails(case)
    H, KV, D, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    R, start = sum(rows), _starts(rows)
    group = [k for k, n in enumerate(rows) for _ in range(n)]
    pages = sum(p // ps for p in prefix) + sum(-(-t // ps) for t in tails)
    ids = (torch.randperm(pages, generator=g, device=DEV) + 1).tolist()         # pages as a pool in use hands them out; page 0 is nobody's
    shared = [[ids.pop() for _ in range(p // ps)] for p in prefix]
    table = [shared[group[r]] + [ids.pop() for _ in range(-(-tails[r] // ps))] for r in range(R)]
    width = max(len(t) for t in table)
    normal = lambda *shape, std=1.0: torch.empty(shape, device=DEV, dtype=dtype).normal_(0.0, std, generator=g)      # noqa: E731
    qkv = normal(R, (H + 2 * KV) * D)                                            # the queries are a view of the projection's rows
    k, v = normal(pages + 1, KV, ps, D), normal(pages + 1, KV, ps, D, std=0.9)
    kv_len = [prefix[group[r]] + tails[r] for r in range(R)]
    meta = SimpleNamespace(decode_segs=_i32(range(R)), seg_q_start=_i32(range(R + 1)), seg_kv_len=_i32(kv_len), table_rows=None, max_pages=width, page_size=ps,
                           block_table=_i32([t + [0] * (width - len(t)) for t in table]), max_kv_len=max(kv_len), shared_start=_i32(start), shared_len=_i32(prefix),
                           max_shared_rows=max(rows), max_shared_len=max(prefix))
    members, place = _members(rows)
    return SimpleNamespace(kind="attention", q=qkv[:, :H * D], k=k, v=v, meta=meta, H=H, KV=KV, D=D, scale=D ** -0.5, members=members, place=place,
                           group=torch.tensor(group, device=DEV), longest=max(prefix), longest_tail=max(tails))


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder, "attention": _prepare_attention}[case["kind"]](case, seed)


# ---------------------------------------------------------------- one pass
def _select_plain(s):
    """Float64 where candidates are ordered: the order of two near ones is a whole number."""
    m = s.logits.amax(1, keepdim=True).double()
    total = (s.logits.double() - m).exp().sum(1, keepdim=True)
    base = s.scores.double()[:, None] - (m + total.log())
    base = torch.where(base.isfinite(), base, -math.inf)
    n = min(s.num, s.logits.shape[1])
    top, token = s.logits.sort(dim=1, descending=True, stable=True)
    top, token = top[:, :n], token[:, :n]
    cand = base + top.double()
    absent = s.members < 0
    grouped = cand[s.members.clamp_min(0)].masked_fill(absent[:, :, None], -math.inf).flatten(1)
    value, at = grouped.sort(dim=1, descending=True, stable=True)
    value, at = value[:, :s.num], at[:, :s.num]
    row = s.members.gather(1, at // n)
    token = token[row, at % n]
    none = value == -math.inf
    row, token = row.masked_fill(none, -1), token.masked_fill(none, -1)
    short = s.num - value.shape[1]
    pad = lambda t, v: torch.nn.functional.pad(t, (0, short), value=v)           # noqa: E731
    return pad(value.float(), -math.inf), pad(row.int(), -1), pad(token.int(), -1)


def _reorder_plain(s):
    source = s.rows[s.parents.long()].long()
    lead = (slice(None),) * s.dim
    for t in s.tensors:
        t[lead + (s.rows.long(),)] = t[lead + (source,)]
    return s.tensors


def _attention_plain(s):
    m, R, KV, D = s.meta, s.q.shape[0], s.KV, s.D
    Hg, ps, (G, B) = s.H // s.KV, s.meta.page_size, s.members.shape
    q = s.q.float().view(R, KV, Hg, D) * s.scale
    # the prefixes: a group's queries together
    n = max(-(-s.longest // ps), 1)
    head = m.block_table[m.shared_start[:-1].long(), :n].long()
    kp, vp = (c[head].float().permute(0, 2, 1, 3, 4).reshape(G, KV, -1, D) for c in (s.k, s.v))
    qg = q[s.members.clamp_min(0)].permute(0, 2, 1, 3, 4).reshape(G, KV, B * Hg, D)
    seen = torch.arange(n * ps, device=q.device)[None, :] < m.shared_len[:, None]
    sp = (qg @ kp.transpose(-1, -2)).masked_fill(~seen[:, None, None, :], -math.inf)
    # the tails
    cols = m.shared_len.long()[s.group][:, None] // ps + torch.arange(-(-s.longest_tail // ps), device=q.device)
    tail = m.block_table.long().gather(1, cols.clamp_max(m.max_pages - 1))
    kt, vt = (c[tail].float().permute(0, 2, 1, 3, 4).reshape(R, KV, -1, D) for c in (s.k, s.v))
    key = m.shared_len.long()[s.group][:, None] + torch.arange(kt.shape[2], device=q.device)
    st = (q @ kt.transpose(-1, -2)).masked_fill(~(key < m.seg_kv_len[:, None])[:, None, None, :], -math.inf)
    # one softmax over both
    by_row = lambda t: t.view(G, KV, B, Hg, -1).permute(0, 2, 1, 3, 4).reshape(G * B, KV, Hg, -1)[s.place]      # noqa: E731
    top = torch.maximum(by_row(sp.amax(-1, keepdim=True)), st.amax(-1, keepdim=True))
    top_g = torch.zeros(G * B, KV, Hg, 1, device=q.device).index_copy(0, s.place, top).view(G, B, KV, Hg, 1).permute(0, 2, 1, 3, 4).reshape(G, KV, B * Hg, 1)
    pp, pt = (sp - top_g).exp(), (st - top).exp()
    total = by_row(pp.sum(-1, keepdim=True)) + pt.sum(-1, keepdim=True)
    return ((by_row(pp @ vp) + pt @ vt) / total).reshape(R, s.H * D).to(s.q.dtype)


def run(state):
    s = state
    if own:
        from mini_inference_b200.ops import get_ops
        ops = get_ops(DEV)
        if s.kind == "select":
            return ops.beam_select(s.logits, s.scores, s.group_start, s.num)
        if s.kind == "reorder":
            ops.reorder_rows(s.tensors, s.rows, s.parents, s.group_start, s.beams, dim=s.dim)
            return s.tensors
        return ops.shared_prefix_attention(s.q, s.k, s.v, s.meta, s.H, s.KV, s.D, s.scale)
    return {"select": _select_plain, "reorder": _reorder_plain, "attention": _attention_plain}[s.kind](s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "select":
        rows = _ints(case["rows"])
        return {"bytes": sum(rows) * (case["vocab"] * 4 + 4) + len(rows) * case["num"] * 12, "flops": 4 * sum(rows) * case["vocab"]}
    if case["kind"] == "reorder":
        if case["form"] == "pages":
            row = case["layers"] * 2 * case["row"] * 2
        else:
            row = sum(4 * case["row"] + 2 * 3 * 301 * (1 + i % 3) + 4 * (1 + i % 3) for i in range(case["layers"]))
        return {"bytes": case["groups"] * (case["moved"] + case["sources"]) * row, "flops": 0}
    rows, prefix, tails = _ints(case["rows"]), _ints(case["prefix"]), _tails(case)
    size = 4 if case["dtype"] == "float32" else 2
    seen = sum(n * p for n, p in zip(rows, prefix)) + sum(tails)
    keys = sum(prefix) + sum(tails)
    return {"bytes": size * case["dim"] * (2 * case["kv_heads"] * keys + 2 * case["heads"] * sum(rows)), "flops": 4 * case["heads"] * case["dim"] * seen}


# ---------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "reorder":                     # copies; whole numbers have no value in 64 bits
        rows, parents, out = s.rows.tolist(), s.parents.tolist(), []
        for t in s.tensors:
            source = list(range(t.shape[s.dim]))
            for r, p in zip(rows, parents):
                source[r] = rows[p]
            out.append(t.double().index_select(s.dim, torch.tensor(source, device=DEV)) if t.is_floating_point() else None)
        return out
    if case["kind"] == "select":
        out = []
        for a, b in zip(s.group_start.tolist(), s.group_start.tolist()[1:]):
            cand = (torch.log_softmax(s.logits[a:b].double(), dim=1) + s.scores[a:b].double()[:, None]).flatten()
            best = torch.full((s.num,), -math.inf, dtype=torch.float64, device=DEV)
            n = min(s.num, cand.numel())
            best[:n] = cand.topk(n).values
            out.append(best)
        return torch.stack(out), None, None
    m, out = s.meta, []
    for r, n in enumerate(m.seg_kv_len.tolist()):     # every row by its own pages alone
        pages = m.block_table[r, :-(-n // m.page_size)].long()
        k, v = (c[pages].double().transpose(1, 2).reshape(-1, s.KV, s.D)[:n].repeat_interleave(s.H // s.KV, dim=1) for c in (s.k, s.v))
        q = s.q[r].double().view(s.H, s.D)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) * s.scale, dim=1)
        out.append(torch.einsum("hn,nhd->hd", p, v).flatten())
    return torch.stack(out)
