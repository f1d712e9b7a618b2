"""Beam search over an engine's model and cache: every beam is a request of its own in the cache (its pages, its state slot), the
steps run all beams as one batch, and after each the beams go on from their parents' caches, which are moved in place. The
reference's engine has no such mode: its sessions go on one token at a time (crates/cellm-sdk/src/lib.rs:227-502)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Sequence

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
    """The cached side of a search: R * K requests in the cache, beam k of prompt r at r * K + k."""

    def __init__(self, engine, prompts, beams: int):
        self.cache, self.runner = engine.cache, engine.runner
        self.R, self.K = len(prompts), beams
        self.prompt_lens = [len(p) for p in prompts]
        self.ids: list[int] = []
        for _ in range(self.R * self.K):
            self.cache.add(engine._next_id)
            self.ids.append(engine._next_id)
            engine._next_id += 1
        dev = self.cache.device
        self.slots = torch.tensor([self.cache.slot(i) for i in self.ids], dtype=torch.int32, device=dev)
        self.starts = torch.tensor(self.prompt_lens, dtype=torch.int32, device=dev)

    def release(self) -> None:
        for i in self.ids:
            self.cache.release(i)

    def hold(self, beam: int, total: int) -> None:
        """Pages for `total` tokens of a beam whose rows will come from another's."""
        if not self.cache.reserve(self.ids[beam], total):
            raise OutOfPages(f"beam search: no pages left for {total} tokens of beam {beam % self.K} of prompt {beam // self.K} "
                             f"(free: {[self.cache.free_pages(g) for g in range(len(self.cache.paged_keys))]})")
        self.cache.commit(self.ids[beam], total)

    def follow(self, parents: torch.Tensor, starts: torch.Tensor) -> None:
        """Every beam goes on from its parent's cache; its rows from `starts` on are moved."""
        for state in self.cache.states:
            ops.reorder_states(state, self.slots, parents, self.runner.err)
        if not self.cache.paged_keys:
            return
        lens = [self.cache.tokens(self.ids[r * self.K]) for r in range(self.R)]
        width = max(1, -(-max(lens) // self.cache.page_size))
        tables = np.full((len(self.cache.paged_keys), len(self.ids), width), -1, dtype=np.int32)
        for g in range(len(self.cache.paged_keys)):
            for b, i in enumerate(self.ids):
                self.cache.block_table(i, g, tables[g, b])
        tables = torch.from_numpy(tables).to(parents.device)
        ends = torch.tensor(lens, dtype=torch.int32, device=parents.device)
        for g, (k, v) in enumerate(zip(self.cache.k_pools, self.cache.v_pools)):
            ops.reorder_pages(k, v, tables[g], starts, ends, parents, self.runner.err)


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
    # the prompts through their first beams, in portions; the others' pages keep step, so that windows give back the same ones
    portion = min(engine.config.prefill_chunk, engine.config.max_batch_tokens)
    rows = []
    for r, prompt in enumerate(prompts):
        for at in range(0, len(prompt), portion):
            part = prompt[at:at + portion]
            last = at + len(part) == len(prompt)
            logits = runner.run([StepEntry(group.ids[r * K], part, [len(part) - 1] if last else [])], limit)
            for k in range(1, K):
                group.hold(r * K + k, at + len(part))
        rows.append(logits.clone())
    scores, parents, tokens = ops.beam_select(torch.cat(rows), torch.zeros((R, 1), device=dev), K)
    # all of a prompt's beams start from the first one's cache, those too that find no continuation yet (a vocabulary of fewer tokens)
    group.follow(torch.zeros_like(parents), torch.zeros_like(group.starts))
    done = tokens == eos if eos is not None else torch.zeros((R, K), dtype=torch.bool, device=dev)
    histories = [[[t] for t in row] for row in tokens.tolist()]
    for _ in range(max_new_tokens - 1):
        if bool((done | (scores == -math.inf)).all()):
            break
        # a finished beam runs along with its last token: what that leaves in its cache nobody reads
        entries = [StepEntry(group.ids[r * K + k], [max(histories[r][k][-1], 0)], [0]) for r in range(R) for k in range(K)]
        logits = runner.run(entries, limit)
        scores, parents, tokens = ops.beam_select(logits, scores, K, done=done)
        group.follow(parents, group.starts)
        was_done = done.gather(1, parents.clamp(min=0).long())
        done = was_done | (tokens == eos) if eos is not None else was_done
        for r, (p_row, t_row, d_row) in enumerate(zip(parents.tolist(), tokens.tolist(), was_done.tolist())):
            histories[r] = [histories[r][p] + ([] if d else [t]) if p >= 0 else [-1] for p, t, d in zip(p_row, t_row, d_row)]
    runner.check()
    out = []
    for row, s_row, d_row in zip(histories, scores.tolist(), done.tolist()):
        found = [BeamOutput(h, s, d) for h, s, d in zip(row, s_row, d_row) if s > -math.inf]
        out.append(sorted(found, key=lambda b: -b.score / len(b.tokens) ** length_penalty))
    return out
