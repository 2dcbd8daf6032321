"""Beam search over the step function: several continuations of a prompt advance together and the best by their summed log-probability survive.

The reference decodes greedily or by temperature only (engine/core/sampler.py:3-11); it has no counterpart of this.  A step
feeds every beam its newest token (one entry each), picks every prompt's best candidates over its beams and the vocabulary on the device
(CudaOps.beam_select) and reads them back: twice as many as beams, more with several end-of-sequence tokens, so that enough go on when some end.  The beams that go on take
over their parents' caches (CacheManager.reorder): full pages by reference, the last page and recurrent states by one copy in place.  Attention over
full contexts reads what all beams of a prompt share once (CudaOps.shared_prefix_attention)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Sequence

import torch

from .batch import StepEntry
from .runner import CacheFull

MAX_BEAMS = 64
MAX_CANDIDATES = 128               # that beam_select gives a group (CudaOps.MAX_CANDIDATES)


@dataclass
class BeamParams:
    num_beams: int = 4
    max_new_tokens: int = 100
    length_penalty: float = 1.0       # a hypothesis of n tokens is ranked by its summed log-probability / n ** length_penalty
    ignore_eos: bool = False          # end-of-sequence tokens are tokens like others

    def __post_init__(self):
        if not 1 <= self.num_beams <= MAX_BEAMS:
            raise ValueError(f"{self.num_beams} beams: between 1 and {MAX_BEAMS} are possible")
        if self.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        if not abs(self.length_penalty) <= 64:
            raise ValueError("length_penalty must be between -64 and 64")
        if abs(self.length_penalty) * math.log(self.max_new_tokens) > 650:      # a rank divides a score by that power: both stay floats
            raise ValueError(f"a length of {self.max_new_tokens} to the power of length_penalty ({self.length_penalty}) is no number")


@dataclass
class Beam:
    """A finished hypothesis: its generated tokens (the end-of-sequence token among them), their summed log-probability, how it ended."""
    tokens: List[int]
    score: float
    rank: float                       # score / len(tokens) ** length_penalty
    finish_reason: str                # "stop" or "length"


class BeamGroup:
    """The beams of one prompt: their tokens and running scores, and the hypotheses that ended.  Host bookkeeping only."""

    def __init__(self, prompt: Sequence[int], params: BeamParams, eos_ids):
        self.prompt, self.params = list(prompt), params
        self.eos_ids = frozenset() if params.ignore_eos else frozenset(eos_ids)
        self.seqs: list = []
        self.tokens: List[List[int]] = [[]]
        self.scores: List[float] = [0.0]
        self.ended: List[Beam] = []
        self.done = False

    def _end(self, tokens, score, reason):
        n = self.params.num_beams
        self.ended.append(Beam(tokens, score, score / len(tokens) ** self.params.length_penalty, reason))
        self.ended.sort(key=lambda b: -b.rank)            # stable: of equals the earlier one stays in front
        del self.ended[n:]

    def advance(self, candidates) -> List[int]:
        """candidates: (score, beam, token), best first, the empty places left out.  Returns the parents of the beams that go on, num_beams of them
        (beams without a candidate keep their own parent and a score of -inf)."""
        n = self.params.num_beams
        live = []
        for rank, (score, beam, token) in enumerate(candidates):
            if token in self.eos_ids:
                if rank < n:                              # an ending counts only where it is among the best n
                    self._end(self.tokens[beam] + [token], score, "stop")
            elif len(live) < n:
                live.append((score, beam, token))
        parents = [b for _, b, _ in live]
        self.tokens, self.scores = [self.tokens[b] + [t] for _, b, t in live], [s for s, _, _ in live]
        while len(parents) < n:
            parents.append(len(parents))
            self.tokens.append(self.tokens[0] if live else [0])
            self.scores.append(-math.inf)
        length = len(self.tokens[0])
        if not live or length >= self.params.max_new_tokens:
            for score, tokens in zip(self.scores, self.tokens):
                if score > -math.inf:
                    self._end(tokens, score, "length")
            self.done = True
        elif len(self.ended) == n:
            # no beam can still overtake the worst of the n that ended: scores only fall, so a rank is at most what the best one has now
            # (by its present length, or by the longest where a longer one ranks higher)
            best, p = max(self.scores), self.params.length_penalty
            self.done = best / (length if p <= 0 else self.params.max_new_tokens) ** p <= self.ended[-1].rank
        return parents


class BeamSearch:
    """Runs groups of beams to their end: as many prompts at a time as the cache has slots and pages for."""

    def __init__(self, llm):
        self.llm, self.cache, self.runner, self.ops = llm, llm.cache, llm.runner, llm.ops
        self._pages = self._slots = 0    # what the admitted groups may still take

    def run(self, prompts, params: BeamParams) -> List[List[Beam]]:
        groups = [BeamGroup(p, params, self.llm.eos_ids) for p in prompts]
        waiting = list(groups)
        while waiting:
            wave = []
            try:
                while waiting and self._admit(waiting[0]):
                    wave.append(waiting.pop(0))
                if not wave:
                    raise CacheFull(f"not enough free cache for {params.num_beams} beams of a prompt of {len(waiting[0].prompt)} tokens and {params.max_new_tokens} more")
                self._run_wave(wave)
            finally:
                for g in wave:
                    self._free(g)
        return [g.ended for g in groups]

    def _admit(self, group) -> bool:
        """A slot per beam, and the pages that the group may come to need beside what the admitted ones hold or may still take."""
        n, p, cache = group.params.num_beams, group.params, self.cache
        pages = cache.pages_for(len(group.prompt)) + n * (cache.pages_for(p.max_new_tokens) + 1)
        if cache.slots.num_free - self._slots < n or len(group.prompt) + p.max_new_tokens > cache.max_pages_per_seq * cache.page_size:
            return False
        if cache.kv_groups and pages + self._pages > cache.free_pages():
            return False
        seq = cache.admit(("beam", id(group), 0))
        if seq is None:
            return False
        group.seqs = [seq]
        self._pages += pages
        self._slots += n - 1
        return True

    def _free(self, group):
        for s in group.seqs:
            if s.alive:
                self.cache.free(s)
        group.seqs = []
        self._pages = self._slots = 0

    def _ensure(self, seq, tokens):
        if not self.cache.ensure(seq, tokens):
            raise CacheFull(f"no pages left for {seq.seq_id!r} to reach {tokens} tokens")

    def _run_wave(self, wave):
        logits = self._prompts(wave)
        for g in wave:                                     # the other beams' slots; they are filled from the first one's
            more = self.cache.fork(g.seqs[0], [("beam", id(g), i) for i in range(1, g.params.num_beams)])
            if more is None:
                raise CacheFull("no slots or pages left for the beams")
            g.seqs += more
        live = wave
        while True:
            moves = self._select(live, logits)
            live = [g for g in live if not g.done]
            if not live:
                return
            self.cache.reorder([(g.seqs, parents) for g, parents in moves if not g.done], self.ops)
            entries = []
            for g in live:
                for seq, tokens in zip(g.seqs, g.tokens):
                    self._ensure(seq, seq.num_tokens + 1)
                    entries.append(StepEntry(seq, [tokens[-1]], [0]))
            logits = self.runner.step(entries, ensure=False)

    def _prompts(self, wave):
        """The prompts, in steps of at most max_batched_tokens tokens; the logits behind each one's last token."""
        budget, logits, entries, used = self.llm.args.max_batched_tokens, {}, [], 0

        def flush():
            nonlocal entries, used
            if entries:
                out = self.runner.step([e for e, _ in entries], ensure=False)
                ends = [g for e, g in entries if e.want]
                for row, g in enumerate(ends):
                    logits[id(g)] = out[row]
            entries, used = [], 0
        for g in wave:
            at = 0
            while at < len(g.prompt):
                if used >= budget:
                    flush()
                n = min(len(g.prompt) - at, budget - used)
                self._ensure(g.seqs[0], at + n)
                last = at + n == len(g.prompt)
                entries.append((StepEntry(g.seqs[0], g.prompt[at:at + n], [n - 1] if last else []), g))
                used += n
                at += n
                if not last:
                    flush()
        flush()
        return torch.stack([logits[id(g)] for g in wave])

    def _select(self, live, logits):
        """Advances every group by its best candidates; returns (group, parents)."""
        starts = [0]
        for g in live:
            starts.append(starts[-1] + len(g.scores))
        # each of n beams can end in any of e ways: with n more candidates, n go on whatever ends
        n, ends = live[0].params.num_beams, sum(0 <= t < logits.shape[1] for t in live[0].eos_ids)
        num, bounds = n * max(2, 1 + ends), starts
        if num > MAX_CANDIDATES:   # of every beam by itself, n and e hold as many that count; they are put in order here, equal values by the lower beam
            num, bounds = n + ends, list(range(starts[-1] + 1))
        dev = logits.device
        # float32 holds what beams are behind their prompt's best one, not a long search's sums: those are kept in 64 bits, here
        tops = [max(g.scores) for g in live]
        host = torch.tensor([s - top for g, top in zip(live, tops) for s in g.scores], dtype=torch.float32)
        start = torch.tensor(bounds, dtype=torch.int32)
        if dev.type == "cuda":
            host, start = host.pin_memory(), start.pin_memory()
        values, rows, tokens = self.ops.beam_select(logits, host.to(dev, non_blocking=True), start.to(dev, non_blocking=True), num)
        out = torch.stack([values.view(torch.int32), rows, tokens]).cpu()              # the step's one device->host sync
        values, rows, tokens = out[0].view(torch.float32).tolist(), out[1].tolist(), out[2].tolist()
        moves = []
        for i, g in enumerate(live):
            lists = range(starts[i], starts[i + 1]) if bounds is not starts else (i,)
            found = [(tops[i] + v, r - starts[i], t) for k in lists for v, r, t in zip(values[k], rows[k], tokens[k]) if r >= 0]
            if len(lists) > 1:
                found.sort(key=lambda c: -c[0])               # stable: lower beams first
            moves.append((g, g.advance(found)))
        return moves
