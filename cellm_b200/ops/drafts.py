"""Trees of drafted tokens: attention of all nodes of a request's tree at once, and which of them stand.

A tree is a run of nodes; node i names its parent by its place in the run: -1 hangs on the request's last committed token, anything
below -1 marks padding (it sees nothing, nobody sees it, its output is zero). A parent stands before its child. Node 0 is usually
the token the last step chose, and the others continue it. A node's position is the request's committed length plus its depth:
that is what its query and key are to be rotated by (`qk_norm_rope` with nkv = 0 does so without writing any page). The nodes' keys
and values stay beside the cache until `accept_drafts` has found which of them are kept."""
from __future__ import annotations

from struct import Struct
from typing import Optional, Sequence

import torch

from ._lib import DTYPE_TAG, dense_ints, fn, launch_packed
from ._state import _SM_COUNT, sm_count

MAX_TREE = 256                     # nodes of a tree (TREE_MAX in draft_tree.cuh)
_TREE_ARGS, _ACCEPT_ARGS = Struct("24qd6q").pack, Struct("28q").pack


def _plan(*sizes) -> int:
    """The native library's plan of a call; from the first call on this name is the library's own function."""
    global _plan
    _plan = fn("attention_tree", "cellm_attention_tree_plan")
    return _plan(*sizes)


def _pitch(t: torch.Tensor, T: int, width: int, dtype, index: int) -> int:
    """The row pitch of `t`, [T, width] or [T, heads, head size] with dense rows of `width` values, in elements; -1: it is none."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not dtype or t.get_device() != index or shape[0] != T:
        return -1
    if len(shape) == 2:
        ok = shape[1] == width and (stride[1] == 1 or width == 1)
    else:
        ok = len(shape) == 3 and shape[1] * shape[2] == width and stride[2] == 1 and (stride[1] == shape[2] or shape[1] == 1)
    return (stride[0] if T > 1 else width) if ok or T == 0 else -1


def attention_tree(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, parents: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                   cu_seqlens: torch.Tensor, ctx_lens: torch.Tensor, block_table: torch.Tensor, tree_lens: Sequence[int], nh: int, scale: float,
                   window: int, err: torch.Tensor, max_ctx: int = 0) -> torch.Tensor:
    """Attention of drafted trees over the paged cache: every node sees its request's committed keys 0 .. ctx_lens[b] - 1 (with a
    `window` > 0 the last `window` positions up to its own) and, among the nodes, its ancestors and itself.

    q [T, nh * hd], k_new and v_new [T, nkv * hd] or [T, nkv, hd]: rows of the nodes, which may be columns of one wider matrix; parents
    int32 [T] (see the module's text); pools [pages, nkv, page size, hd]; request b owns nodes cu_seqlens[b] .. cu_seqlens[b + 1], at
    most 256, and `tree_lens` is the host's copy of their numbers. `max_ctx`: the longest context if the host knows it (0: what the
    block table can name). float32 or bfloat16, heads of up to 256. Returns [T, nh * hd]; rows of no tree hold nothing of meaning. A row of K or V
    that is not finite may reach every node of its tree. Nothing is read or written of padding and of page entries that no node sees. A
    page out of range that a node does see is reported in `err`, and its keys and values are zeros. Scores, maxima and sums are 32-bit;
    in bfloat16 with heads of 32, 64, 96 or 128 the softmax's weights are rounded to bfloat16 before they meet the values, an error of up to
    2^-8 of the weighted values' magnitudes beside the output's own rounding."""
    dtype, index, shape, table, T, B = q.dtype, q.get_device(), k_pool.shape, block_table.shape, q.shape[0], len(tree_lens)
    if index < 0 or dtype not in DTYPE_TAG or len(shape) != 4:
        raise ValueError("attention_tree: float32 or bfloat16 rows on the GPU over pools [pages, kv heads, page size, head size]")
    pages, nkv, page_size, hd = shape
    if nkv <= 0 or nh <= 0 or nh % nkv or not 0 < hd <= 256:
        raise ValueError(f"attention_tree: {nh} heads over {nkv} of {hd}: whole groups of heads of up to 256 only")
    if v_pool.shape != shape or k_pool.dtype is not dtype or v_pool.dtype is not dtype or k_pool.get_device() != index or v_pool.get_device() != index \
            or not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise ValueError(f"attention_tree: dense pools of {dtype} and one shape on {q.device}")
    q_ld, k_ld, v_ld = _pitch(q, T, nh * hd, dtype, index), _pitch(k_new, T, nkv * hd, dtype, index), _pitch(v_new, T, nkv * hd, dtype, index)
    if q_ld < 0 or k_ld < 0 or v_ld < 0:
        raise ValueError(f"attention_tree: q [{T}, {nh * hd}], k_new and v_new [{T}, {nkv * hd}] of {dtype} on {q.device} with dense rows (got "
                         + ", ".join(f"{tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}" for t in (q, k_new, v_new)) + ")")
    if not dense_ints(index, parents, cu_seqlens, ctx_lens, block_table, err):
        raise ValueError(f"attention_tree: parents, cu_seqlens, ctx_lens, block_table and err must be dense int32 on {q.device}")
    if parents.numel() != T or cu_seqlens.numel() != B + 1 or ctx_lens.numel() != B or len(table) != 2 or table[0] != B or err.numel() < 1:
        raise ValueError(f"attention_tree: parents [{T}], cu_seqlens [{B + 1}], ctx_lens [{B}], block_table [{B}, entries] and an error word")
    most = max(tree_lens) if B else 0
    if B and (most > MAX_TREE or min(tree_lens) < 0 or sum(tree_lens) > T):
        raise ValueError(f"attention_tree: trees of 0 to {MAX_TREE} nodes, {T} in all (got {list(tree_lens)})")
    if window < 0 or max_ctx < 0:
        raise ValueError("attention_tree: window and max_ctx must not be negative")
    out = q.new_empty((T, nh * hd))
    if most == 0:
        return out
    entries, tag = table[1], DTYPE_TAG[dtype]
    keys = entries * page_size
    if 0 < max_ctx < keys:
        keys = max_ctx
    if 0 < window < keys:
        keys = window
    plan = _plan(B, most, nh, nkv, hd, keys + most, tag, _SM_COUNT.get(index) or sm_count(index))
    nsplit, parts, part_o, part_ml = plan & 0xff, plan >> 8 & 0xff, 0, 0
    if parts:
        outputs = parts * T * nh * hd + 1 & ~1                         # (what follows them is read in pairs)
        ws = parents.new_empty(outputs + parts * T * nh * 2)           # of 32-bit words: the pieces' outputs, then maxima and sums
        part_o = ws.data_ptr()
        part_ml = part_o + 4 * outputs
    launch_packed("attention_tree", "attention_tree", index,
                  _TREE_ARGS(out.data_ptr(), part_o, part_ml, q.data_ptr(), q_ld, k_new.data_ptr(), k_ld, v_new.data_ptr(), v_ld, parents.data_ptr(), k_pool.data_ptr(),
                             v_pool.data_ptr(), cu_seqlens.data_ptr(), ctx_lens.data_ptr(), block_table.data_ptr(), entries, B, T, most, pages, page_size, nh, nkv, hd,
                             scale, window, nsplit, parts, plan >> 16, tag, err.data_ptr()), 2 if parts else 1)
    return out


def _layers(new: torch.Tensor, pool: torch.Tensor, T: int, index: int):
    """Bytes between items and between nodes of `new` [items, T, heads, size] beside its pool [items, pages, heads, page size, size], and
    bytes of a head's row; None where the two do not fit. Either may lack its first axis."""
    shape, stride, own = new.shape, new.stride(), pool.shape
    if len(shape) == 3:
        shape, stride = (1, *shape), (0, *stride)
    if len(own) == 4:
        own = (1, *own)
    if len(shape) != 4 or len(own) != 5 or new.dtype is not pool.dtype or new.get_device() != index or pool.get_device() != index or not pool.is_contiguous():
        return None
    if shape[0] != own[0] or shape[1] != T or shape[2] != own[2] or shape[3] != own[4]:
        return None
    if T and own[0] and ((stride[3] != 1 and shape[3] > 1) or (stride[2] != shape[3] and shape[2] > 1)):
        return None
    e = new.element_size()
    return (stride[0] * e if own[0] > 1 else 0), (stride[1] * e if T > 1 else 0), shape[3] * e, own


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
    index, T, B = tokens.get_device(), tokens.numel(), cu_seqlens.numel() - 1
    if index < 0 or longest < 1 or not dense_ints(index, tokens, parents, choices, cu_seqlens, err):
        raise ValueError("accept_drafts: dense int32 arrays on one GPU and a longest path of at least one node")
    if parents.numel() != T or choices.numel() != T or B < 0 or err.numel() < 1:
        raise ValueError("accept_drafts: tokens, parents and choices of one length, cu_seqlens [requests + 1], an error word")
    if (k_new is None) != (k_pool is None) or (v_new is None) != (v_pool is None) or (v_new is not None and k_new is None):
        raise ValueError("accept_drafts: rows and pool of the keys (and of the values) together")
    rows = (0,) * 10
    where = (0,) * 7
    if k_new is not None:
        if ctx_lens is None or block_table is None or not dense_ints(index, ctx_lens, block_table) or ctx_lens.numel() != B or block_table.dim() != 2 \
                or block_table.shape[0] != B:
            raise ValueError(f"accept_drafts: rows are written behind ctx_lens [{B}] on the pages of block_table [{B}, entries], dense int32 on {tokens.device}")
        k = _layers(k_new, k_pool, T, index)
        if v_new is None:
            v = (0, 0, 0, None)
        elif (v_new.shape == k_new.shape and v_new.stride() == k_new.stride() and v_pool.shape == k_pool.shape and v_new.dtype is v_pool.dtype is k_pool.dtype
              and v_new.get_device() == index and v_pool.get_device() == index and v_pool.is_contiguous()):
            v = k                                                              # laid out alike
        else:
            v = _layers(v_new, v_pool, T, index)
        if k is None or v is None or (v_new is not None and v[3][:4] != k[3][:4]):
            raise ValueError("accept_drafts: k_new and v_new [items, T, kv heads, head size], a node's heads side by side, of the type of their dense pools [items, pages, "
                             f"kv heads, page size, head size] (got {[tuple(t.shape) for t in (k_new, v_new, k_pool, v_pool) if t is not None]})")
        items, pages, nkv, page_size, _ = k[3]
        rows = (k_new.data_ptr(), k[0], k[1], k[2], k_pool.data_ptr()) + ((v_new.data_ptr(), v[0], v[1], v[2], v_pool.data_ptr()) if v_new is not None else (0,) * 5)
        where = (ctx_lens.data_ptr(), block_table.data_ptr(), block_table.shape[1], items, nkv, pages, page_size)
    path = tokens.new_empty((B, longest))
    count = tokens.new_empty(B) if k_new is None or ctx_lens.dim() != 1 else torch.empty_like(ctx_lens)
    after = torch.empty_like(count)
    if B:
        launch_packed("candidates", "accept_drafts", index,
                      _ACCEPT_ARGS(count.data_ptr(), path.data_ptr(), after.data_ptr(), tokens.data_ptr(), parents.data_ptr(), choices.data_ptr(), cu_seqlens.data_ptr(),
                                   B, T, longest, *rows, *where, err.data_ptr()))
    return count, path, after
