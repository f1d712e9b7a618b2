"""What the operators over drafted trees and beams refuse, on the CPU: the C entry points before anything is launched, and the Python
ones before they ask for memory; and which host rules choose their launches."""
import ctypes

import pytest
import torch

from cellm_b200 import ops
from cellm_b200.ops import _lib

BUF = ctypes.create_string_buffer(4096)
A = (ctypes.addressof(BUF) + 255) & ~255        # a 256-byte aligned address that no refused call reads
DTYPE, SIZE, ALIGN, ARG = -1, -2, -3, -4


def call(library, name, *args):
    return _lib.fn(library, name)(*args)


def test_attention_of_trees():
    def tree(out=A, part=None, q=A, parents=A, cu=A, T=8, B=2, most=5, page=16, nh=4, nkv=2, hd=64, window=0, nsplit=1, parts=0, dtype=1, err=A):
        return call("attention_tree", "cellm_attention_tree", out, part, part, q, nh * hd, A, nkv * hd, A, nkv * hd, parents, A, A, cu, A, A, 4, B, T, most, 8, page, nh, nkv,
                    hd, 0.125, window, nsplit, parts, 1, dtype, err, None)
    assert tree(dtype=2) == DTYPE and tree(dtype=-1) == DTYPE
    for bad in (dict(nh=5), dict(nkv=0), dict(nh=0), dict(hd=0), dict(hd=257), dict(page=0), dict(most=257), dict(window=-1), dict(nsplit=0), dict(nsplit=65, part=A), dict(parts=-1)):
        assert tree(**bad) == SIZE, bad
    assert tree(nsplit=2, parts=2) == ARG and tree(parts=2, part=A + 4) == ALIGN and tree(out=None) == ARG and tree(parents=None) == ARG and tree(err=None) == ARG
    assert tree(T=0) == 0 and tree(B=0) == 0 and tree(most=0) == 0


def test_plans_of_attention_of_trees():
    """Pieces, pieces in the workspace, tcgen05 or not: by the rows of a tree and the keys before them."""
    def plan(B, most, keys, nh=32, nkv=8, hd=64, dtype=1):
        p = call("attention_tree", "cellm_attention_tree_plan", B, most, nh, nkv, hd, keys, dtype, 148)
        return p & 0xff, p >> 8 & 0xff, p >> 16
    n, parts, tc = plan(1, 8, 508)
    assert tc == 0 and 1 < n <= 8 and parts == 0                   # a cluster, no workspace
    assert plan(16, 25, 4121)[2] == 1 and plan(8, 16, 4096)[2] == 1 and plan(8, 16, 1024)[2] == 0 and plan(8, 4, 30000)[2] == 0
    assert plan(8, 25, 4121, dtype=0)[2] == 0 and plan(8, 25, 4121, hd=128)[2] == 0 and plan(8, 25, 4121, nh=70, nkv=1)[2] == 0       # (70 of 128 rows)
    for B in (1, 3, 8, 64):
        for most in (1, 5, 16, 63, 256):
            for keys in (1, 100, 5000, 100000):
                for hd in (32, 64, 96, 128, 200):
                    for dtype in (0, 1):
                        n, parts, tc = plan(B, most, keys, hd=hd, dtype=dtype)
                        assert 1 <= n <= 64 and parts == (n if n > (1 if tc else 8) else 0)
    assert plan(64, 63, 100)[0] == 1                                # enough blocks without cutting


def test_acceptance():
    def accept(count=A, tokens=A, B=2, T=8, longest=4, k=A, k_item=256, k_row=64, k_bytes=32, k_pool=A, v=None, v_pool=None, v_bytes=32, ctx=A, items=1, nkv=2, pages=4, page=16):
        return call("candidates", "cellm_accept_drafts", count, A, A, tokens, A, A, A, B, T, longest, k, k_item, k_row, k_bytes, k_pool, v, 256, 64, v_bytes, v_pool, ctx, A, 4,
                    items, nkv, pages, page, A, None)
    for bad in (dict(longest=0), dict(B=65536), dict(T=-1), dict(items=-1), dict(nkv=0), dict(pages=0), dict(page=0), dict(k_bytes=0)):
        assert accept(**bad) == SIZE, bad
    for bad in (dict(count=None), dict(tokens=None), dict(k=None), dict(k_pool=None), dict(ctx=None), dict(v=A), dict(v=A, v_pool=A, v_bytes=0)):
        assert accept(**bad) == ARG, bad
    assert accept(k=A + 1) == ALIGN and accept(k_bytes=33) == ALIGN and accept(k_row=63) == ALIGN
    assert accept(B=0) == 0


def test_selection_and_reordering():
    def select(out=A, logits=A, ld=100, V=100, R=2, K=3, keep=4, scores=A, pad=0, dtype=0, sums=A):
        return call("candidates", "cellm_beam_select", out, A, A, A, sums, logits, ld, V, R, K, keep, scores, None, pad, dtype, 148, None)
    assert select(dtype=2) == DTYPE
    for bad in (dict(V=0), dict(K=0), dict(K=33), dict(keep=0), dict(keep=65), dict(ld=99), dict(pad=100), dict(pad=-1), dict(R=2 ** 29), dict(V=2 ** 30, ld=2 ** 30)):
        assert select(**bad) == SIZE, bad
    assert select(out=None) == ARG and select(scores=None) == ARG and select(sums=A + 8) == ALIGN and select(logits=A + 2) == ALIGN and select(R=0) == 0

    def states(state=A, slots=A, R=2, K=3, items=1, n=8, size=64):
        return call("candidates", "cellm_reorder_states", state, slots, A, R, K, items, n, size, A, None)
    for bad in (dict(K=0), dict(K=33), dict(n=0), dict(items=65536), dict(R=65536)):
        assert states(**bad) == SIZE, bad
    assert states(state=None) == ARG and states(slots=None) == ARG and states(size=63) == ALIGN and states(state=A + 1) == ALIGN
    assert states(R=0) == 0 and states(items=0) == 0 and states(size=0) == 0

    def pages(pool=A, table=A, stride=4, R=2, K=3, items=1, n=8, nkv=2, page=16, row=64, v=None, v_row=0):
        return call("candidates", "cellm_reorder_pages", pool, row, v, v_row, table, stride, A, A, A, R, K, items, n, nkv, page, 148, A, None)
    for bad in (dict(K=0), dict(K=33), dict(n=0), dict(nkv=0), dict(page=0), dict(stride=0), dict(items=65536), dict(R=65536), dict(row=0), dict(v=A), dict(page=2 ** 30)):
        assert pages(**bad) == SIZE, bad
    assert pages(pool=None) == ARG and pages(table=None) == ARG and pages(row=63) == ALIGN and pages(v=A, v_row=63) == ALIGN and pages(v=A + 1, v_row=64) == ALIGN
    assert pages(R=0) == 0 and pages(items=0) == 0


def test_tensors_on_the_host_are_refused():
    """None of these may reach a kernel: the first tensor does not lie on a GPU."""
    i = torch.zeros(4, dtype=torch.int32)
    rows, pool = torch.zeros(4, 64), torch.zeros(3, 1, 16, 64)
    with pytest.raises(ValueError, match="attention_tree"):
        ops.attention_tree(rows, rows, rows, i, pool, pool, i[:2], i[:1], i[:1].view(1, 1), [4], 1, 0.125, 0, i[:1])
    with pytest.raises(ValueError, match="accept_drafts"):
        ops.accept_drafts(i, i, i, i[:2], 3, i[:1])
    with pytest.raises(ValueError, match="beam_select"):
        ops.beam_select(rows, torch.zeros(2, 2), 4)
    with pytest.raises(ValueError, match="reorder_states"):
        ops.reorder_states(pool, i, i.view(2, 2), i[:1])
    with pytest.raises(ValueError, match="reorder_pages"):
        ops.reorder_pages(pool, pool, i.view(4, 1), i[:2], i[:2], i.view(2, 2), i[:1])
