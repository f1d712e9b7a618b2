"""Beam search over an engine's model and cache: every beam that goes on is a request of its own in the cache (its pages, its state slot),
the steps run these beams as one batch, and after each the beams go on from their parents' caches, which are moved in place. The
reference's engine has no such mode: its sessions go on one token at a time (crates/cellm-sdk/src/lib.rs:227-502)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from .. import ops
from ..cache.manager import OutOfPages
from ..ops.beams import MAX_BEAMS
from .step import StepEntry


@dataclass
class BeamOutput:
    tokens: list[int]           # generated, the end-of-sequence token among them where it was chosen
    score: float                # sum of the tokens' log probabilities
    finished: bool              # it ended with the end-of-sequence token


class _Beams:
    """The cached side of a search: up to K requests of the cache a prompt, its places. A beam that goes on has one; which, does not matter.
    One that has ended, and one that was never found, has none: nobody reads what its cache would hold."""

    def __init__(self, engine, prompts, beams: int):
        self.engine, self.cache, self.runner = engine, engine.cache, engine.runner
        self.R, self.K = len(prompts), beams
        self.prompt_lens = [len(p) for p in prompts]
        self.portion = min(engine.config.prefill_chunk, engine.config.max_batch_tokens)
        self.ids: list[list[Optional[int]]] = [[None] * beams for _ in prompts]      # of the places
        self.slots = [[-1] * beams for _ in prompts]                                  # of the places; -1: it has none
        self.place: list[list[Optional[int]]] = [[None] * beams for _ in prompts]    # of the beams

    def take(self, r: int, place: int) -> None:
        request = self.engine._next_id
        self.slots[r][place] = self.cache.add(request)
        self.engine._next_id += 1
        self.ids[r][place] = request

    def give_back(self, r: int, place: int) -> None:
        if self.ids[r][place] is not None:
            self.cache.release(self.ids[r][place])
            self.ids[r][place], self.slots[r][place] = None, -1

    def tokens(self, r: int) -> int:
        """What is cached of each of a prompt's beams; 0 where none goes on."""
        return next((self.cache.tokens(i) for i in self.ids[r] if i is not None), 0)

    def release(self) -> None:
        for r in range(self.R):
            for place in range(self.K):
                self.give_back(r, place)

    def request(self, r: int, beam: int) -> int:
        return self.ids[r][self.place[r][beam]]

    def hold(self, r: int, place: int, total: int) -> None:
        """Pages for `total` tokens of a place whose rows will come from another's, portion by portion, so that windows give back the same ones."""
        at = self.cache.tokens(self.ids[r][place])
        while at < total:
            at = min(at + self.portion, total)
            if not self.cache.reserve(self.ids[r][place], at):
                raise OutOfPages(f"beam search: no pages left for {at} tokens of a beam of prompt {r} "
                                 f"(free: {[self.cache.free_pages(g) for g in range(len(self.cache.paged_keys))]})")
            self.cache.commit(self.ids[r][place], at)

    def follow(self, parents: Sequence[Sequence[int]]) -> None:
        """Beam k of prompt r goes on from the cache of beam parents[r][k]; a parent of -1: it does not go on, and its cache is given back.
        A beam stays in its parent's place where it is the first to ask for it; the others' rows are moved."""
        moves = [[-1] * self.K for _ in parents]                # by place
        news = [[] for _ in parents]
        for r, row in enumerate(parents):
            old, self.place[r] = self.place[r], [None] * self.K
            stay: dict[int, int] = {}
            for k, p in enumerate(row):
                if p >= 0:
                    stay.setdefault(old[p], k)
            for place, k in stay.items():
                self.place[r][k] = place
            free = [x for x in range(self.K) if x not in stay]
            free.sort(key=lambda x: self.ids[r][x] is None)      # places that hold a cache first
            for k, p in enumerate(row):
                if p >= 0 and self.place[r][k] is None:
                    place = self.place[r][k] = free.pop(0)
                    moves[r][place] = old[p]
                    if self.ids[r][place] is None:
                        news[r].append(place)
            for place in free:
                self.give_back(r, place)
        if all(p < 0 for row in moves for p in row):
            return
        lens = [self.tokens(r) for r in range(self.R)]
        for r, places in enumerate(news):
            for place in places:
                self.take(r, place)
                self.hold(r, place, lens[r])
        self._move(moves, [0 if new else n for new, n in zip(news, self.prompt_lens)], lens)

    def _move(self, moves, starts, lens) -> None:
        dev = self.cache.device
        flat = [i for row in self.ids for i in row]
        slots = [s for row in self.slots for s in row]
        if -1 in slots:                                          # (places that hold nothing: nothing of theirs is moved)
            spare = iter(set(range(self.cache.num_slots)) - set(slots))
            slots = [s if s >= 0 else next(spare) for s in slots]
        width = max(1, -(-max(lens) // self.cache.page_size))
        tables = np.full((len(self.cache.paged_keys), len(flat), width), -1, dtype=np.int32)
        for g in range(len(self.cache.paged_keys)):
            for b, i in enumerate(flat):
                if i is not None:
                    self.cache.block_table(i, g, tables[g, b])
        n, R = len(flat), self.R
        numbers = torch.from_numpy(np.concatenate([np.asarray(x, dtype=np.int32).reshape(-1) for x in (moves, slots, starts, lens, tables)])).to(dev)
        parents, slots, starts, ends, rest = numbers[:n].view(R, self.K), numbers[n:2 * n], numbers[2 * n:2 * n + R], numbers[2 * n + R:2 * n + 2 * R], numbers[2 * n + 2 * R:]
        for state in self.cache.states:
            ops.reorder_states(state, slots, parents, self.runner.err)
        for g, (k, v) in enumerate(zip(self.cache.k_pools, self.cache.v_pools)):
            ops.reorder_pages(k, v, rest[g * n * width:(g + 1) * n * width].view(n, width), starts, ends, parents, self.runner.err)


def beam_search(engine, prompts: Sequence[Sequence[int]], beams: int, max_new_tokens: int, length_penalty: float,
                stop_eos: bool) -> list[list[BeamOutput]]:
    """See Engine.beam_search."""
    plan, config, cache = engine.plan, engine.config, engine.cache
    prompts = [[int(t) for t in p] for p in prompts]
    R, K, V = len(prompts), int(beams), plan.vocab_size
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError(f"beam search takes 1 to {MAX_BEAMS} beams")
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be at least 1")
    if any(not p for p in prompts):
        raise ValueError("a prompt needs at least one token")
    bad = [t for p in prompts for t in p if not 0 <= t < V]
    if bad:
        raise ValueError(f"token id {bad[0]} outside the vocabulary of {V}")
    longest = max((len(p) for p in prompts), default=0) + max_new_tokens - 1          # (the last token is not run)
    if longest > plan.max_positions:
        raise ValueError(f"{longest} tokens exceed the model's {plan.max_positions} positions")
    if engine.has_unfinished():
        raise RuntimeError("beam search needs the engine's cache to itself: requests are unfinished")
    if R * K > min(cache.free_slots, config.max_batch_tokens):
        raise ValueError(f"{R} prompts of {K} beams need as many state slots and tokens a step "
                         f"(max_num_seqs leaves {cache.free_slots}, max_batch_tokens is {config.max_batch_tokens})")
    if not R:
        return []
    eos = plan.eos_token_id if stop_eos else None
    group = _Beams(engine, prompts, K)
    try:
        return _search(engine, group, prompts, K, max_new_tokens, length_penalty, eos)
    finally:
        group.release()


def _search(engine, group: _Beams, prompts, K: int, max_new_tokens: int, length_penalty: float, eos):
    R, dev, runner, limit = len(prompts), engine.cache.device, engine.runner, engine.max_layers
    rows = []
    for r, prompt in enumerate(prompts):                # in portions, through the first beam
        group.take(r, 0)
        group.place[r][0] = 0
        for at in range(0, len(prompt), group.portion):
            part = prompt[at:at + group.portion]
            last = at + len(part) == len(prompt)
            logits = runner.run([StepEntry(group.request(r, 0), part, [len(part) - 1] if last else [])], limit)
        rows.append(logits.clone())
    scores, parents, tokens = ops.beam_select(torch.cat(rows), torch.zeros((R, 1), device=dev), K)
    histories: list[list[list[int]]] = [[[]] for _ in prompts]
    done = [[False] for _ in prompts]
    for at in range(max_new_tokens):
        s_rows, p_rows, t_rows = scores.tolist(), parents.tolist(), tokens.tolist()
        was_done = [[p >= 0 and row[p] for p in p_row] for row, p_row in zip(done, p_rows)]
        histories = [[row[p] + ([] if d else [t]) if p >= 0 else [] for p, t, d in zip(p_row, t_row, d_row)]
                     for row, p_row, t_row, d_row in zip(histories, p_rows, t_rows, was_done)]
        done = [[d or (eos is not None and t == eos) for t, d in zip(t_row, d_row)] for t_row, d_row in zip(t_rows, was_done)]
        going = [[p if not d and s > -math.inf else -1 for p, d, s in zip(p_row, d_row, s_row)] for p_row, d_row, s_row in zip(p_rows, done, s_rows)]
        live = [r * K + k for r in range(R) for k in range(K) if going[r][k] >= 0]
        if at + 1 == max_new_tokens or not live:
            break
        group.follow(going)
        logits = runner.run([StepEntry(group.request(b // K, b % K), [histories[b // K][b % K][-1]], [0]) for b in live], limit)
        over = None
        if len(live) < R * K:                           # rows of beams that do not go on are not looked at
            at_rows = torch.tensor(live, dtype=torch.long).to(dev)
            over = torch.ones(R * K, dtype=torch.bool, device=dev).index_fill_(0, at_rows, False).view(R, K)
            logits = logits.new_empty((R * K, logits.shape[1])).index_copy_(0, at_rows, logits)
        scores, parents, tokens = ops.beam_select(logits, scores, K, done=over)
    runner.check()
    out = []
    for row, s_row, d_row in zip(histories, s_rows, done):
        found = [BeamOutput(h, s, d) for h, s, d in zip(row, s_row, d_row) if s > -math.inf]
        out.append(sorted(found, key=lambda b: -b.score / len(b.tokens) ** length_penalty))
    return out
