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
