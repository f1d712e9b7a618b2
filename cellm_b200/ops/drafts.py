"""Trees of drafted tokens: attention of all nodes of a request's tree at once, and which of them stand.

A tree is a run of nodes; node i names its parent by its place in the run: -1 hangs on the request's last committed token, anything
below -1 marks padding (it sees nothing, nobody sees it, its output is zero). A parent stands before its child. Node 0 is usually
the token the last step chose, and the others continue it. A node's position is the request's committed length plus its depth:
that is what its query and key are to be rotated by (`qk_norm_rope` with nkv = 0 does so without writing any page). The nodes' keys
and values stay beside the cache until `accept_drafts` has found which of them are kept."""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from ._lib import DTYPE_TAG, fn, launch, ptr, require_ints
from ._state import sm_count

MAX_TREE = 256                     # nodes of a tree (TREE_MAX in draft_tree.cuh)


def _rows(name: str, what: str, t: torch.Tensor, T: int, width: int, like: torch.Tensor) -> int:
    """The row pitch of `t` [T, width], or [T, heads, head size] with dense heads, in elements."""
    inner = t.stride(-1) == 1 and (t.dim() == 2 or (t.dim() == 3 and t.stride(1) == t.shape[2]))
    if t.dtype != like.dtype or t.device != like.device or t.shape[0] != T or t.numel() != T * width or (T and not inner):
        raise ValueError(f"{name}: {what} must be [{T}, {width}] rows of {like.dtype} on {like.device} with dense rows "
                         f"(got {tuple(t.shape)}, strides {t.stride()}, {t.dtype}, {t.device})")
    return t.stride(0) if T > 1 else width


def attention_tree(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, parents: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                   cu_seqlens: torch.Tensor, ctx_lens: torch.Tensor, block_table: torch.Tensor, tree_lens: Sequence[int], nh: int, scale: float,
                   window: int, err: torch.Tensor, max_ctx: int = 0) -> torch.Tensor:
    """Attention of drafted trees over the paged cache: every node sees its request's committed keys 0 .. ctx_lens[b] - 1 (with a
    `window` > 0 the last `window` positions up to its own) and, among the nodes, its ancestors and itself.

    q [T, nh * hd], k_new and v_new [T, nkv * hd] or [T, nkv, hd]: rows of the nodes, which may be columns of one wider matrix; parents
    int32 [T] (see the module's text); pools [pages, nkv, page size, hd]; request b owns nodes cu_seqlens[b] .. cu_seqlens[b + 1], at
    most 256, and `tree_lens` is the host's copy of their numbers. `max_ctx`: the longest context if the host knows it (0: what the
    block table can name). float32 or bfloat16, heads of up to 256. Returns [T, nh * hd]. A row of K or V that is not finite may reach
    every node of its tree. Nothing is read or written of padding and of page entries that no node sees."""
    name = "attention_tree"
    if not q.is_cuda or k_pool.dim() != 4 or q.dtype not in DTYPE_TAG:
        raise ValueError(f"{name}: float32 or bfloat16 rows on the GPU over pools [pages, kv heads, page size, head size]")
    pages, nkv, page_size, hd = k_pool.shape
    T, B, device = q.shape[0], len(tree_lens), q.device
    if nkv <= 0 or nh <= 0 or nh % nkv or not 0 < hd <= 256:
        raise ValueError(f"{name}: {nh} heads over {nkv} of {hd}: whole groups of heads of up to 256 only")
    for pool in (k_pool, v_pool):
        if pool.dtype != q.dtype or pool.device != device or not pool.is_contiguous() or pool.shape != k_pool.shape:
            raise ValueError(f"{name}: dense pools of {q.dtype} and one shape on {device}")
    q_ld, k_ld, v_ld = (_rows(name, what, t, T, w, q) for what, t, w in (("q", q, nh * hd), ("k_new", k_new, nkv * hd), ("v_new", v_new, nkv * hd)))
    require_ints(name, device, parents=parents, cu_seqlens=cu_seqlens, ctx_lens=ctx_lens, block_table=block_table, err=err)
    if parents.numel() != T or cu_seqlens.numel() != B + 1 or ctx_lens.numel() != B or block_table.dim() != 2 or block_table.shape[0] != B or err.numel() < 1:
        raise ValueError(f"{name}: parents [{T}], cu_seqlens [{B + 1}], ctx_lens [{B}], block_table [{B}, entries] and an error word")
    most = max(tree_lens, default=0)
    if most > MAX_TREE or min(tree_lens, default=0) < 0 or sum(tree_lens) > T:
        raise ValueError(f"{name}: trees of 0 to {MAX_TREE} nodes, {T} in all (got {list(tree_lens)})")
    if window < 0 or max_ctx < 0:
        raise ValueError(f"{name}: window and max_ctx must not be negative")
    out = torch.empty((T, nh * hd), dtype=q.dtype, device=device)
    if most == 0:
        return out
    entries = block_table.shape[1]
    keys = min(max_ctx or entries * page_size, entries * page_size)
    keys = min(keys, window) if window else keys
    nsplit = fn("attention_tree", "cellm_attention_tree_pieces")(B, most, nh, nkv, hd, keys + most, DTYPE_TAG[q.dtype], sm_count(device))
    part_o = part_ml = None
    if nsplit > 1:
        ws = torch.empty(nsplit * T * nh * (hd + 2), dtype=torch.float32, device=device)
        part_o, part_ml = ws.data_ptr(), ws.data_ptr() + 4 * nsplit * T * nh * hd
    launch("attention_tree", name, q, ptr(out), part_o, part_ml, ptr(q), q_ld, ptr(k_new), k_ld, ptr(v_new), v_ld, ptr(parents), ptr(k_pool), ptr(v_pool),
           ptr(cu_seqlens), ptr(ctx_lens), ptr(block_table), entries, B, T, most, pages, page_size, nh, nkv, hd, float(scale), int(window), nsplit,
           DTYPE_TAG[q.dtype], ptr(err), kernels=2 if nsplit > 1 else 1)
    return out


def _draft_rows(new: Optional[torch.Tensor], pool: Optional[torch.Tensor], T: int, what: str):
    """Pointer, bytes between items and nodes, bytes of a head's row, pointer to the pool: of one of keys and values."""
    if new is None:
        return None, 0, 0, 0, None
    if new.dim() == 3:
        new = new.unsqueeze(0)
    items, pages, nkv, page_size, width = pool.shape
    if new.dim() != 4 or new.shape != (items, T, nkv, width) or new.dtype != pool.dtype or new.device != pool.device or not pool.is_contiguous():
        raise ValueError(f"accept_drafts: {what}_new must be [{items}, {T}, {nkv}, {width}] {pool.dtype} beside its dense pool {tuple(pool.shape)} "
                         f"(got {tuple(new.shape)} {new.dtype})")
    if new.numel() and (new.stride(3) != 1 or (nkv > 1 and new.stride(2) != width)):
        raise ValueError(f"accept_drafts: a node's {what} heads must lie side by side")
    e = new.element_size()
    return new.data_ptr(), new.stride(0) * e if items > 1 else 0, new.stride(1) * e if T > 1 else 0, width * e, pool.data_ptr()


def accept_drafts(tokens: torch.Tensor, parents: torch.Tensor, choices: torch.Tensor, cu_seqlens: torch.Tensor, longest: int, err: torch.Tensor,
                  k_new: Optional[torch.Tensor] = None, v_new: Optional[torch.Tensor] = None, k_pool: Optional[torch.Tensor] = None,
                  v_pool: Optional[torch.Tensor] = None, ctx_lens: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None):
    """Which nodes of drafted trees stand. tokens int32 [T]: what the nodes drafted; choices int32 [T]: what the model chose after each
    (an arg-max or a draw); parents, cu_seqlens as for `attention_tree`. Node 0 of a tree stands; then, node after node, the child
    whose token is the choice after the node (the first among equals), up to `longest` nodes. Of a tree without nodes, or whose first
    is padding, none does.

    Returns int32 (count [B], path [B, longest]: the standing nodes' places in their tree, -1 behind them, next [B]: the choice after
    the last one, -1 where there is none). With the nodes' keys and values k_new and v_new [items, T, nkv, hd] (or without the first
    axis) and the pools [items, pages, nkv, page size, hd] (or without it) the standing nodes' rows are written to places ctx_lens[b],
    ctx_lens[b] + 1, ... of the request's pages; v_new and v_pool None: keys alone."""
    name = "accept_drafts"
    device = tokens.device
    if not tokens.is_cuda or longest < 1:
        raise ValueError(f"{name}: arrays on the GPU and a longest path of at least one node")
    require_ints(name, device, tokens=tokens, parents=parents, choices=choices, cu_seqlens=cu_seqlens, err=err)
    T, B = tokens.numel(), cu_seqlens.numel() - 1
    if parents.numel() != T or choices.numel() != T or B < 0 or err.numel() < 1:
        raise ValueError(f"{name}: tokens, parents and choices of one length, cu_seqlens [requests + 1], an error word")
    items = nkv = pages = page_size = entries = 0
    if (k_new is None) != (k_pool is None) or (v_new is None) != (v_pool is None) or (v_new is not None and k_new is None):
        raise ValueError(f"{name}: rows and pool of the keys (and of the values) together")
    if k_new is not None:
        if ctx_lens is None or block_table is None:
            raise ValueError(f"{name}: rows are written behind ctx_lens on the pages of block_table")
        require_ints(name, device, ctx_lens=ctx_lens, block_table=block_table)
        if ctx_lens.numel() != B or block_table.dim() != 2 or block_table.shape[0] != B or k_pool.device != device:
            raise ValueError(f"{name}: ctx_lens [{B}] and block_table [{B}, entries] on {device}")
        k_pool = k_pool.unsqueeze(0) if k_pool.dim() == 4 else k_pool
        v_pool = v_pool.unsqueeze(0) if v_pool is not None and v_pool.dim() == 4 else v_pool
        if k_pool.dim() != 5 or (v_pool is not None and v_pool.shape[:4] != k_pool.shape[:4]):
            raise ValueError(f"{name}: pools [items, pages, kv heads, page size, head size] of one shape but for the head size")
        items, pages, nkv, page_size, _ = k_pool.shape
        entries = block_table.shape[1]
    k, v = _draft_rows(k_new, k_pool, T, "k"), _draft_rows(v_new, v_pool, T, "v")
    out = torch.empty((B, longest + 2), dtype=torch.int32, device=device).view(-1)
    count, after, path = out[:B], out[B:2 * B], out[2 * B:].view(B, longest)
    launch("candidates", name, tokens, ptr(count), ptr(path), ptr(after), ptr(tokens), ptr(parents), ptr(choices), ptr(cu_seqlens), B, T, int(longest), *k, *v,
           ptr(ctx_lens), ptr(block_table), entries, items, nkv, pages, page_size, ptr(err))
    return count, path, after
