"""Plain statements of beam search's operators in 64 bits, as TorchRefOps has the other kernels: what the CUDA kernels are tested against, and what
lets the engine's beam search run on the CPU inside the tests."""
from __future__ import annotations

import math

import torch

from tests.ref_ops import TorchRefOps


def beam_select64(logits, scores, group_start, num):
    """(values float64, rows, tokens) [G, num], by sorting every candidate of a group."""
    starts, V = group_start.tolist(), logits.shape[1]
    values = torch.full((len(starts) - 1, num), -math.inf, dtype=torch.float64)
    rows, tokens = torch.full(values.shape, -1, dtype=torch.int32), torch.full(values.shape, -1, dtype=torch.int32)
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        found = []
        for r in range(a, b):
            x = logits[r].double().cpu() + 0.0
            base = float(scores[r].double() - torch.logsumexp(x, 0).to(scores.device))
            if not math.isfinite(base):
                continue
            order = torch.sort(x, descending=True, stable=True).indices[:num]
            found += [(-(base + float(x[t])), r, -float(x[t]), int(t)) for t in order if x[t] > -math.inf]
        for i, (v, r, _, t) in enumerate(sorted(found)[:num]):
            values[g, i], rows[g, i], tokens[g, i] = -v, r, t
    return values, rows, tokens


def reorder_rows_plain(tensors, rows, parents, group_start, dim=0):
    for t in tensors:
        lead = (slice(None),) * dim
        old = t.clone()
        for a, b in zip(group_start.tolist(), group_start.tolist()[1:]):
            for i in range(a, b):
                p = int(parents[i])
                if a <= p < b and 0 <= int(rows[i]) < t.shape[dim] and 0 <= int(rows[p]) < t.shape[dim]:
                    t[lead + (int(rows[i]),)] = old[lead + (int(rows[p]),)]


class BeamRefOps(TorchRefOps):
    def beam_select(self, logits, scores, group_start, num):
        v, r, t = beam_select64(logits, scores, group_start, num)
        return v.float().to(logits.device), r.to(logits.device), t.to(logits.device)

    def reorder_rows(self, tensors, rows, parents, group_start, most, dim=0):
        reorder_rows_plain(tensors, rows, parents, group_start, dim)


def shared_prefix_attention64(q, k_cache, v_cache, meta, H, KV, D, scale):
    """(output, sum of weights times |values|, largest sum of |q k| scale) of the entries' rows in float64, by row: keys below its group's shared length by
    the pages of the group's first row that has them all, the others by its own."""
    R, ps, Hg = meta.decode_segs.shape[0], meta.page_size, H // KV
    starts, shared = meta.shared_start.tolist(), meta.shared_len.tolist()
    segs, toks, lens = meta.decode_segs.tolist(), meta.seg_q_start.tolist(), meta.seg_kv_len.tolist()
    rows = list(range(len(lens))) if getattr(meta, "table_rows", None) is None else meta.table_rows.tolist()
    table, k64, v64 = meta.block_table.cpu(), k_cache.cpu().double(), v_cache.cpu().double()
    out = torch.zeros(q.shape[0], H * D, dtype=torch.float64)
    size, reach = torch.zeros_like(out), 0.0
    for r in range(R):
        n, tok = lens[segs[r]], toks[segs[r]]
        if n <= 0:
            continue
        g = next((g for g in range(len(shared)) if starts[g] <= r < starts[g + 1]), None)
        key = torch.arange(n)
        own = table[rows[segs[r]]][key // ps].long()
        if g is not None:
            holds = next((i for i in range(starts[g], starts[g + 1]) if lens[segs[i]] >= shared[g]), starts[g])
            own = torch.where(key < shared[g], table[rows[segs[holds]]][key // ps].long(), own)
        k, v = k64[own, :, key % ps], v64[own, :, key % ps]                       # [n, KV, D]
        qr = q[tok].cpu().double().view(KV, Hg, D)
        s = torch.einsum("khd,nkd->khn", qr, k) * scale
        reach = max(reach, float((torch.einsum("khd,nkd->khn", qr.abs(), k.abs()) * scale).max()))
        w = torch.softmax(s, dim=-1)
        out[tok] = torch.einsum("khn,nkd->khd", w, v).reshape(-1)
        size[tok] = torch.einsum("khn,nkd->khd", w, v.abs()).reshape(-1)
    return out, size, reach


def _shared_prefix_attention(self, q, k_cache, v_cache, meta, H, KV, D, scale):
    return shared_prefix_attention64(q, k_cache, v_cache, meta, H, KV, D, scale)[0].to(q.device, q.dtype)


BeamRefOps.shared_prefix_attention = _shared_prefix_attention
