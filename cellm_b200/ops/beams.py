"""Beam search: the best continuations of a request's beams, and the beams' cached state in their new order."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import DTYPE_TAG, fn, launch, ptr, require_ints

MAX_BEAMS, MAX_KEEP = 32, 64       # (as in beams.cu)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, keep: int, done: Optional[torch.Tensor] = None, pad: int = 0):
    """The `keep` best continuations (beam k, token v) of each request, by scores[r, k] + log softmax(logits[r * K + k])[v], best first
    and equal ones by (k, v). logits [R * K, V] float32 or bfloat16 (rows may be strided), scores float32 [R, K], K and `keep` up to 32
    and 64. done [R, K] bool: a finished beam offers itself alone, with token `pad`, at its score (its logits are not looked at).
    A beam with score -inf and a token with logit -inf (a NaN counts as one) are never chosen; logits of +inf have no meaning here.
    Scores are compared in 64 bits; the sums behind them carry about 2^-25.

    Returns (scores float32, parents int32, tokens int32), each [R, keep]; where a request has fewer continuations, -inf and -1."""
    name = "beam_select"
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in DTYPE_TAG or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"{name}: float32 or bfloat16 logits [requests * beams, V] on the GPU, rows dense")
    device, (rows, V) = logits.device, logits.shape
    if scores.dtype != torch.float32 or scores.device != device or scores.dim() != 2 or not scores.is_contiguous() or scores.numel() != rows:
        raise ValueError(f"{name}: dense float32 scores [requests, beams] for {rows} rows of logits on {device} (got {tuple(scores.shape)} {scores.dtype})")
    R, K = scores.shape
    if not 0 < K <= MAX_BEAMS or not 0 < keep <= MAX_KEEP or V < 1 or not 0 <= pad < V:
        raise ValueError(f"{name}: up to {MAX_BEAMS} beams, up to {MAX_KEEP} kept and a padding token of the vocabulary (got {K}, {keep}, {pad} of {V})")
    if done is not None and (done.dtype != torch.bool or done.device != device or done.shape != scores.shape or not done.is_contiguous()):
        raise ValueError(f"{name}: done must be dense bool {tuple(scores.shape)} on {device}")
    out_scores = torch.empty((R, keep), dtype=torch.float32, device=device)
    picked = torch.empty((2, R, keep), dtype=torch.int32, device=device)
    if R:
        parts = fn("candidates", "cellm_beam_parts")(V)
        # the rows' sums (two 64-bit numbers a part), then their lanes' maxima (32 floats a part)
        ws = torch.empty(rows * parts * 36, dtype=torch.float32, device=device)
        at = ws.data_ptr()
        launch("candidates", name, logits, ptr(out_scores), picked.data_ptr(), picked.data_ptr() + 4 * R * keep, at + 16 * rows * parts, at, ptr(logits),
               logits.stride(0) if rows > 1 else V, V, R, K, int(keep), ptr(scores), ptr(done), int(pad), DTYPE_TAG[logits.dtype], kernels=2)
    return out_scores, picked[0], picked[1]


def _beams(name: str, parents: torch.Tensor, err: torch.Tensor):
    if parents.dim() != 2 or not parents.is_cuda or not 0 < parents.shape[1] <= MAX_BEAMS or err.numel() < 1:
        raise ValueError(f"{name}: parents int32 [requests, beams] with up to {MAX_BEAMS} beams on the GPU, and an error word")
    require_ints(name, parents.device, parents=parents, err=err)
    return parents.shape


def reorder_states(state: torch.Tensor, slot_ids: torch.Tensor, parents: torch.Tensor, err: torch.Tensor) -> None:
    """In place: beam k of request r goes on from the state of beam parents[r, k]. state [items, slots, ...] dense (as the cache manager
    keeps a group's states), of any element type; slot_ids int32 [requests * beams] (or [requests, beams]), a slot for each beam and no
    slot for two. A parent of -1, or the beam itself, leaves its state as it is. A parent or slot out of range is reported in `err` and
    the beam left alone."""
    name = "reorder_states"
    R, K = _beams(name, parents, err)
    require_ints(name, parents.device, slot_ids=slot_ids)
    if state.dim() < 2 or state.device != parents.device or not state.is_contiguous() or slot_ids.numel() != R * K or state.element_size() % 2:
        raise ValueError(f"{name}: a dense state [items, slots, ...] of elements of 2, 4 or 8 bytes on {parents.device} and {R * K} slots")
    items, slots = state.shape[:2]
    if state.numel() == 0 or R == 0:
        return
    launch("candidates", name, state, ptr(state), ptr(slot_ids), ptr(parents), R, K, items, slots, state.numel() // (items * slots) * state.element_size(), ptr(err))


def reorder_pages(k_pool: torch.Tensor, v_pool: Optional[torch.Tensor], block_table: torch.Tensor, starts: torch.Tensor, ends: torch.Tensor,
                  parents: torch.Tensor, err: torch.Tensor) -> None:
    """In place: rows starts[r] .. ends[r] - 1 of beam k of request r become those of beam parents[r, k]. Pools [items, pages, kv heads,
    page size, head size] (or without the first axis; v_pool None: keys alone); block_table int32 [requests * beams, entries], every beam
    on pages of its own; what lies before `starts` (the prompt) is the same for all beams of a request and stays. A parent of -1, or the
    beam itself, leaves the rows as they are, an entry of -1 (a page given back) the rows on it. A parent, page or row out of range
    is reported in `err` and passed over."""
    name = "reorder_pages"
    R, K = _beams(name, parents, err)
    device = parents.device
    require_ints(name, device, block_table=block_table, starts=starts, ends=ends)
    if block_table.dim() != 2 or block_table.shape[0] != R * K or starts.numel() != R or ends.numel() != R:
        raise ValueError(f"{name}: block_table [{R * K}, entries], starts [{R}] and ends [{R}]")
    pools = [p for p in (k_pool, v_pool) if p is not None]
    for p in pools:
        if p.dim() not in (4, 5) or p.device != device or not p.is_contiguous() or p.element_size() % 2 or p.shape[:-1] != k_pool.shape[:-1]:
            raise ValueError(f"{name}: dense pools [items, pages, kv heads, page size, head size] of elements of 2, 4 or 8 bytes on {device}, alike but for the head size")
    if R == 0 or block_table.shape[1] == 0:
        return
    for p in pools:
        items = p.shape[0] if p.dim() == 5 else 1
        pages, nkv, page_size, width = p.shape[-4:]
        if p.numel():
            launch("candidates", name, p, ptr(p), ptr(block_table), block_table.shape[1], ptr(starts), ptr(ends), ptr(parents), R, K, items, pages, nkv, page_size,
                   width * p.element_size(), ptr(err))
