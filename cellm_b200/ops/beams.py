"""Beam search: the best continuations of a request's beams, and the beams' cached state in their new order."""
from __future__ import annotations

from struct import Struct
from typing import Optional

import torch

from ._lib import DTYPE_TAG, dense_ints, fn, launch_packed
from ._state import _SM_COUNT, sm_count

MAX_BEAMS, MAX_KEEP, MAX_VOCAB = 32, 64, 1 << 24       # (as in beams.cu)
_SELECT_ARGS, _STATES_ARGS, _PAGES_ARGS = Struct("16q").pack, Struct("9q").pack, Struct("17q").pack


def beam_select(logits: torch.Tensor, scores: torch.Tensor, keep: int, done: Optional[torch.Tensor] = None, pad: int = 0):
    """The `keep` best continuations (beam k, token v) of each request, by scores[r, k] + log softmax(logits[r * K + k])[v], best first
    and equal ones by (k, v). logits [R * K, V] float32 or bfloat16 (rows may be strided; V up to 2^24), scores float32 [R, K], K and `keep` up
    to 32 and 64. done [R, K] bool: a finished beam offers itself alone, with token `pad`, at its score (its logits are not looked at).
    A beam with score -inf and a token with logit -inf (a NaN counts as one) are never chosen; logits of +inf have no meaning here.
    Scores are compared in 64 bits; the log-sums behind them are good to 3e-7, mostly to 2^-25.

    Returns (scores float32, parents int32, tokens int32), each [R, keep]; where a request has fewer continuations, -inf and -1."""
    index, shape, stride, pair = logits.get_device(), logits.shape, logits.stride(), scores.shape
    if index < 0 or len(shape) != 2 or logits.dtype not in DTYPE_TAG or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("beam_select: float32 or bfloat16 logits [requests * beams, V] on the GPU, rows dense")
    rows, V = shape
    if len(pair) != 2 or pair[0] * pair[1] != rows or scores.dtype is not torch.float32 or scores.get_device() != index or not scores.is_contiguous():
        raise ValueError(f"beam_select: dense float32 scores [requests, beams] for {rows} rows of logits on {logits.device} (got {tuple(pair)} {scores.dtype})")
    R, K = pair
    if not 0 < K <= MAX_BEAMS or not 0 < keep <= MAX_KEEP or not 0 < V <= MAX_VOCAB or not 0 <= pad < V:
        raise ValueError(f"beam_select: up to {MAX_BEAMS} beams, up to {MAX_KEEP} kept and a padding token of the vocabulary (got {K}, {keep}, {pad} of {V})")
    if done is not None and (done.dtype is not torch.bool or done.get_device() != index or done.shape != pair or not done.is_contiguous()):
        raise ValueError(f"beam_select: done must be dense bool {tuple(pair)} on {logits.device}")
    best = scores.new_empty((R, keep))
    parents = torch.empty_like(best, dtype=torch.int32)
    tokens = torch.empty_like(parents)
    if R:
        parts = fn("candidates", "cellm_beam_parts")(V)
        # the rows' sums (32 bytes a part), then their lanes' maxima (32 floats a part)
        ws = scores.new_empty(rows * parts * 40)
        at = ws.data_ptr()
        launch_packed("candidates", "beam_select", index,
                      _SELECT_ARGS(best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), at + 32 * rows * parts, at, logits.data_ptr(), stride[0] if rows > 1 else V, V,
                                   R, K, keep, scores.data_ptr(), 0 if done is None else done.data_ptr(), pad, DTYPE_TAG[logits.dtype],
                                   _SM_COUNT.get(index) or sm_count(index)), 2)
    return best, parents, tokens


def reorder_states(state: torch.Tensor, slot_ids: torch.Tensor, parents: torch.Tensor, err: torch.Tensor) -> None:
    """In place: beam k of request r goes on from the state of beam parents[r, k]. state [items, slots, ...] dense (as the cache manager
    keeps a group's states), of any element type; slot_ids int32 [requests * beams] (or [requests, beams]), a slot for each beam and no
    slot for two. A parent of -1, or the beam itself, leaves its state as it is. A parent or slot out of range is reported in `err` and
    the beam left alone."""
    index, shape, pair = parents.get_device(), state.shape, parents.shape
    if index < 0 or len(pair) != 2 or not 0 < pair[1] <= MAX_BEAMS or not dense_ints(index, parents, slot_ids, err) or err.numel() < 1:
        raise ValueError(f"reorder_states: dense int32 parents [requests, beams] with up to {MAX_BEAMS} beams, slots and an error word on one GPU")
    R, K = pair
    e = state.element_size()
    if len(shape) < 2 or state.get_device() != index or not state.is_contiguous() or slot_ids.numel() != R * K or e % 2:
        raise ValueError(f"reorder_states: a dense state [items, slots, ...] of elements of 2, 4 or 8 bytes on {parents.device} and {R * K} slots")
    n = state.numel()
    if n and R:
        launch_packed("candidates", "reorder_states", index,
                      _STATES_ARGS(state.data_ptr(), slot_ids.data_ptr(), parents.data_ptr(), R, K, shape[0], shape[1], n // (shape[0] * shape[1]) * e, err.data_ptr()))


def reorder_pages(k_pool: torch.Tensor, v_pool: Optional[torch.Tensor], block_table: torch.Tensor, starts: torch.Tensor, ends: torch.Tensor,
                  parents: torch.Tensor, err: torch.Tensor) -> None:
    """In place: rows starts[r] .. ends[r] - 1 of beam k of request r become those of beam parents[r, k]. Pools [items, pages, kv heads,
    page size, head size] (or without the first axis; v_pool None: keys alone); block_table int32 [requests * beams, entries], every beam
    on pages of its own; what lies before `starts` (the prompt) is the same for all beams of a request and stays. A parent of -1, or the
    beam itself, leaves the rows as they are, an entry of -1 (a page given back) the rows on it. A parent, page or row out of range
    is reported in `err` and passed over."""
    index, pair, table = parents.get_device(), parents.shape, block_table.shape
    if index < 0 or len(pair) != 2 or not 0 < pair[1] <= MAX_BEAMS or not dense_ints(index, parents, block_table, starts, ends, err) or err.numel() < 1:
        raise ValueError(f"reorder_pages: dense int32 parents [requests, beams] with up to {MAX_BEAMS} beams, block_table, starts, ends and an error word on one GPU")
    R, K = pair
    if len(table) != 2 or table[0] != R * K or starts.numel() != R or ends.numel() != R:
        raise ValueError(f"reorder_pages: block_table [{R * K}, entries], starts [{R}] and ends [{R}]")
    own = k_pool.shape[:-1]
    pools = (k_pool,) if v_pool is None else (k_pool, v_pool)
    for p in pools:
        if len(own) not in (3, 4) or p.shape[:-1] != own or p.get_device() != index or not p.is_contiguous() or p.element_size() % 2:
            raise ValueError("reorder_pages: dense pools [items, pages, kv heads, page size, head size] of elements of 2, 4 or 8 bytes, alike but for the head size, "
                             f"on {parents.device}")
    if R == 0 or table[1] == 0 or k_pool.numel() == 0:
        return
    k, v = k_pool.data_ptr(), 0 if v_pool is None else v_pool.data_ptr()
    launch_packed("candidates", "reorder_pages", index,
                  _PAGES_ARGS(k, k_pool.shape[-1] * k_pool.element_size(), v, v_pool.shape[-1] * v_pool.element_size() if v else 0, block_table.data_ptr(), table[1],
                              starts.data_ptr(), ends.data_ptr(), parents.data_ptr(), R, K, own[0] if len(own) == 4 else 1, own[-3], own[-2], own[-1],
                              _SM_COUNT.get(index) or sm_count(index), err.data_ptr()))
