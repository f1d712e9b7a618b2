"""Attention of drafted trees and the acceptance of drafts against plain 64-bit restatements: trees of one node and of the most
there may be, padding, contexts of none, of one token and across pages and blocks, windows shorter than a tree, odd head sizes,
strided rows; a step of drafting as a program runs it; refusals and bad pages."""
import numpy as np
import pytest
import torch

import plain_candidates as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def err_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def make_tree(r, n, padding=0, chain=False):
    if chain:
        return list(range(-1, n - 1))
    parents = [-1] + [int(r.randint(max(-1, i - 9), i)) for i in range(1, n)]
    for i in range(n - padding, n):
        parents[i] = -2 - int(r.randint(0, 3))
    return parents[:n]


def make(r, dtype, lens, ctxs, nh, nkv, hd, page, padding=0, chain=False, wide=True, spare=0):
    g = torch.Generator().manual_seed(int(r.randint(1 << 30)))
    T = sum(lens)
    need = [-(-c // page) + spare for c in ctxs]
    order = r.permutation(sum(need) + 2).tolist()
    table = np.full((len(lens), max(need) + 1), -1)
    for b, n in enumerate(need):
        table[b, :n] = [order.pop() for _ in range(n)]
    shape = (sum(need) + 2, nkv, page, hd)
    # rows that no node sees are not numbers: pages nobody owns, and what lies behind a context on its last page
    pools = []
    for _ in range(2):
        p = torch.full(shape, float("nan"))
        for b, c in enumerate(ctxs):
            for j in range(c):
                p[table[b, j // page], :, j % page] = torch.randn(nkv, hd, generator=g)
        pools.append(p.to(dtype).to(DEV))
    rows = torch.randn(T, (nh + 2 * nkv) * hd + (8 if wide else 0), generator=g).to(dtype).to(DEV)
    parents = [p for n in lens for p in make_tree(r, n, min(padding, n - 1) if n else 0, chain)]
    at = 0
    for n in lens:
        for i in range(n):
            if plain.lineage(parents[at:at + n], i) is None:
                rows[at + i, nh * hd:] = float("nan")
        at += n
    cut = lambda a, b: rows[:, a * hd:b * hd] if wide else rows[:, a * hd:b * hd].contiguous()
    return dict(q=cut(0, nh), k_new=cut(nh, nh + nkv), v_new=cut(nh + nkv, nh + 2 * nkv), parents=parents, k=pools[0], v=pools[1], lens=lens,
                ctxs=ctxs, table=table, cu=ints(np.concatenate([[0], np.cumsum(lens)])), nh=nh)


def run(x, window=0, max_ctx=0, scale=None, err=None):
    from cellm_b200 import ops
    e = err_word() if err is None else err
    hd = x["k"].shape[3]
    out = ops.attention_tree(x["q"], x["k_new"], x["v_new"], ints(x["parents"]), x["k"], x["v"], x["cu"], ints(x["ctxs"]), ints(x["table"]), x["lens"], x["nh"],
                             hd ** -0.5 if scale is None else scale, window, e, max_ctx=max_ctx)
    if err is None:
        assert e.item() == 0
    return out


def check(x, out, window=0, scale=None):
    hd = x["k"].shape[3]
    ref, mass, size, count = plain.attention_tree(x["q"], x["k_new"], x["v_new"], x["parents"], x["k"], x["v"], x["lens"], x["ctxs"], x["table"], x["nh"],
                                                  hd ** -0.5 if scale is None else scale, window)
    got = out.double().cpu().view(ref.shape)
    # 32 bits: a score is off by (hd + 2) half steps of the sum of its products' magnitudes, a weight by that (twice: in the
    # denominator too) and a few steps of the exponential, a sum by half a step a key and a few for the merge of pieces
    rel = 2 * (hd + 2) * 2.0 ** -24 * size + (2 * count + 24) * 2.0 ** -24
    if out.dtype == torch.bfloat16:
        rel = rel + 2.0 ** -8                          # the weights, rounded to bfloat16
    bound = rel.unsqueeze(2) * mass + (2.0 ** -8 * ref.abs() if out.dtype == torch.bfloat16 else 2.0 ** -24 * ref.abs()) * 1.01 + 1e-30
    worst = ((got - ref).abs() / bound).max() if ref.numel() else torch.tensor(0.0)
    assert torch.isfinite(got).all() and float(worst) <= 1.0, f"{float(worst)} times the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,page", [(64, 16), (32, 8), (128, 64), (96, 16), (64, 128), (40, 16), (17, 3), (256, 16), (200, 5)])
@pytest.mark.parametrize("nh,nkv", [(4, 1), (6, 2), (3, 3)])
def test_attention_of_trees(dtype, hd, page, nh, nkv):
    r = np.random.RandomState(hd * 7 + page + nh)
    x = make(r, dtype, [1, 7, 0, 23, 12], [0, 1, 5, 64, 131], nh, nkv, hd, page, padding=2)
    check(x, run(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 2, 5, 40, 64, 1000])
@pytest.mark.parametrize("hd", [64, 128])
def test_windows(dtype, window, hd):
    """Windows shorter than a tree is deep, shorter and longer than the contexts; pages in front of them were given back."""
    r = np.random.RandomState(window + hd)
    x = make(r, dtype, [20, 9, 33], [200, 3, 70], 4, 2, hd, 16, chain=window < 5)
    out = run(x, window)
    check(x, out, window)
    for b, c in enumerate(x["ctxs"]):
        x["table"][b, :max(0, c - window + 1) // 16] = -1
    assert torch.equal(run(x, window), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,nh,nkv,hd", [(256, 2, 1, 64), (255, 1, 1, 64), (128, 8, 2, 64), (65, 12, 4, 64), (200, 4, 2, 128), (130, 3, 1, 32), (40, 40, 1, 64)])
def test_large_trees(dtype, nodes, nh, nkv, hd):
    r = np.random.RandomState(nodes)
    x = make(r, dtype, [nodes, 3, nodes - 1], [77, 300, 0], nh, nkv, hd, 16, padding=5)
    check(x, run(x))
    x = make(r, dtype, [nodes], [129], nh, nkv, hd, 16, chain=True)
    check(x, run(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("nodes", [1, 5, 70])
def test_long_contexts_are_cut_into_pieces(dtype, hd, nodes):
    r = np.random.RandomState(hd + nodes)
    x = make(r, dtype, [nodes, nodes], [3001, 1900], 4, 2, hd, 32, spare=20)
    out = run(x)
    check(x, out)
    check(x, run(x, max_ctx=3001))


@pytest.mark.parametrize("nodes,nh,nkv", [(9, 8, 2), (16, 4, 1), (33, 4, 2), (7, 12, 4), (32, 32, 8)])
@pytest.mark.parametrize("window", [0, 2500])
def test_small_trees_behind_long_contexts(nodes, nh, nkv, window):
    """Few rows on the wide tiles: both tiles of a CTA hold the same rows and take the blocks of keys in turn, an odd and an even
    number of them, one alone for a context without keys."""
    r = np.random.RandomState(nodes)
    x = make(r, torch.bfloat16, [nodes, nodes, nodes], [2600, 0, 4099], nh, nkv, 64, 16, padding=1)
    out = run(x, window)
    check(x, out, window)


def test_rows_may_be_dense_or_columns_and_other_trees_do_not_matter():
    r = np.random.RandomState(3)
    x = make(r, torch.bfloat16, [9, 30], [100, 40], 8, 2, 64, 16)
    out = run(x)
    y = dict(x, q=x["q"].contiguous(), k_new=x["k_new"].contiguous().view(-1, 2, 64), v_new=x["v_new"].contiguous().view(-1, 2, 64))
    assert torch.equal(run(y), out)
    first = dict(x, lens=[9], ctxs=[100], table=x["table"][:1], parents=x["parents"][:9], cu=ints([0, 9]), **{k: x[k][:9] for k in ("q", "k_new", "v_new")})
    check(first, run(first))


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(scale):
    r = np.random.RandomState(5)
    x = make(r, torch.float32, [12], [90], 4, 2, 64, 16)
    check(x, run(x, scale=scale), scale=scale)
    x = make(r, torch.bfloat16, [12, 40], [90, 10], 4, 2, 64, 16)
    check(x, run(x, scale=scale), scale=scale)


def test_nothing_to_do_and_empty_trees():
    r = np.random.RandomState(6)
    x = make(r, torch.bfloat16, [0, 0], [4, 9], 4, 2, 64, 16)
    assert run(x).shape == (0, 4 * 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_pages_and_trees_are_reported_and_left_out(dtype):
    r = np.random.RandomState(7)
    x = make(r, dtype, [6, 20], [100, 50], 4, 2, 64, 16)
    x["parents"] = make_tree(r, 6) + make_tree(r, 20)
    good = run(x)
    for bad in (-1, 10 ** 6):
        y = dict(x, table=x["table"].copy())
        y["table"][1, 0] = bad
        e = err_word()
        out = run(y, err=e)
        assert e.item() == 2 and torch.equal(out[:6], good[:6])
    e = err_word()
    run(dict(x, parents=x["parents"][:6] + [-1, 1] + x["parents"][8:]), err=e)            # node 1 hangs on itself
    assert e.item() == 32
    e = err_word()
    run(dict(x, table=x["table"][:, :2]), err=e)                                          # a context longer than its row of the table
    assert e.item() == 2


def with_zeros(x, bad):
    """The same trees with zeros on entries bad[b] of their requests' tables."""
    pools = {z: x[z].clone() for z in "kv"}
    for b, entries in enumerate(bad):
        for z in "kv":
            pools[z][[x["table"][b, e] for e in entries]] = 0.0
    return dict(x, **pools)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,nh,nkv,hd,page", [(6, 4, 2, 64, 16), (6, 4, 2, 128, 16), (13, 3, 1, 40, 5), (5, 2, 1, 256, 16), (70, 2, 1, 64, 16), (20, 8, 2, 64, 16),
                                                  (40, 4, 1, 64, 128), (50, 6, 2, 64, 8)])
@pytest.mark.parametrize("ctxs", [[100, 50, 37], [400, 1, 300]])
def test_bad_pages_count_as_zeros(dtype, nodes, nh, nkv, hd, page, ctxs):
    """Keys and values of a page that is none are zeros, in all of the kernels: the first, a middle one and the last page, all pages of a
    request, a page in every second place; the trees beside them as without."""
    check_bad_pages(np.random.RandomState(nodes + page + ctxs[0]), dtype, nodes, nh, nkv, hd, page, ctxs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,nh,nkv,hd", [(9, 8, 2, 64), (2, 2, 1, 128), (3, 1, 1, 48)])
def test_bad_pages_in_front_of_pieces(dtype, nodes, nh, nkv, hd):
    check_bad_pages(np.random.RandomState(nodes), dtype, nodes, nh, nkv, hd, 16, [2600, 130, 2100])


def check_bad_pages(r, dtype, nodes, nh, nkv, hd, page, ctxs):
    x = make(r, dtype, [nodes] * 3, ctxs, nh, nkv, hd, page)
    good = run(x)
    last = [-(-c // page) - 1 for c in ctxs]
    for bad in ([{0}, set(), set()], [{last[0] // 2, last[0]}, set(), {0, last[2]}], [set(), set(range(last[1] + 1)), set(range(0, last[2], 2))]):
        y = dict(x, table=x["table"].copy())
        for b, entries in enumerate(bad):
            for i, e in enumerate(sorted(entries)):
                y["table"][b, e] = (-1, x["k"].shape[0], 10 ** 6, -2 ** 31)[i % 4]
        e = err_word()
        out = run(y, err=e)
        assert e.item() == 2
        check(with_zeros(x, bad), out)
        for b in range(3):
            if not bad[b]:
                assert torch.equal(out[b * nodes:(b + 1) * nodes], good[b * nodes:(b + 1) * nodes])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,hd", [(6, 64), (6, 128), (6, 40), (70, 64)])
def test_a_bad_page_inside_a_window(dtype, nodes, hd):
    """Every node's window holds the whole page, and begins inside another."""
    x = make(np.random.RandomState(nodes + hd), dtype, [nodes], [100], 4, 2, hd, 16)
    x["parents"] = [-1] + [0] * (nodes - 1)
    y = dict(x, table=x["table"].copy())
    y["table"][0, 4] = -1                               # keys 64 .. 79; the nodes see those from 52 or 53 on
    e = err_word()
    out = run(y, 49, err=e)
    assert e.item() == 2
    check(with_zeros(x, [{4}]), out, 49)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,hd", [(6, 64), (6, 128), (6, 40), (70, 64)])
@pytest.mark.parametrize("entry", [-2, -3, -2 ** 31, 2 ** 31 - 1])
def test_every_page_that_is_none_is_reported(dtype, nodes, hd, entry):
    x = make(np.random.RandomState(nodes + hd), dtype, [nodes], [100], 4, 2, hd, 16)
    for at in (0, 3, 6):
        y = dict(x, table=x["table"].copy())
        y["table"][0, at] = entry
        e = err_word()
        check(with_zeros(x, [{at}]), run(y, err=e))
        assert e.item() == 2
    y = dict(x, table=x["table"].copy())
    y["table"][0, 0] = entry                                # in front of the window: nothing of it is looked at
    check(x, run(y, 60), 60)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("nodes,window", [(12, 0), (12, 20), (40, 0), (40, 20), (140, 20)])
def test_what_a_node_does_not_see_has_no_weight(dtype, hd, nodes, window):
    """Keys and values near the type's largest, finite, of nodes on other branches and of keys in front of a window: the outputs of the
    nodes that do not see them are what they are with zeros there, bit for bit."""
    r = np.random.RandomState(nodes + hd + window)
    x = make(r, dtype, [nodes], [100], 4, 2, hd, 16)
    x["parents"] = [-1] + [0] * (nodes - 1)
    big = [i for i in range(1, nodes) if i % 5 == 2 or i % 16 == 1]             # (some at every place of a run of 16)
    seen_by = set(big)
    outs = []
    for value in (0.0, 0.99 * torch.finfo(dtype).max):
        y = dict(x, k_new=x["k_new"].clone(), v_new=x["v_new"].clone(), k=x["k"].clone(), v=x["v"].clone())
        for i in big:
            y["k_new"][i], y["v_new"][i] = value, -value
        if window:                                          # key 81 stands in node 0's window alone
            y["k"][x["table"][0, 5], :, 1], y["v"][x["table"][0, 5], :, 1] = value, value
        outs.append(run(y, window))
    others = [i for i in range(1 if window else 0, nodes) if i not in seen_by]
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[1][others], outs[0][others])


def test_a_captured_call_follows_its_inputs():
    r = np.random.RandomState(8)
    x = make(r, torch.bfloat16, [9, 14], [700, 300], 8, 2, 64, 16)
    from cellm_b200 import ops
    ins = dict(parents=ints(x["parents"]), ctx=ints(x["ctxs"]), table=ints(x["table"]), err=err_word())
    call = lambda: ops.attention_tree(x["q"], x["k_new"], x["v_new"], ins["parents"], x["k"], x["v"], x["cu"], ins["ctx"], ins["table"], x["lens"], 8, 0.125, 0, ins["err"])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
        with torch.cuda.graph(other, stream=s):
            second = call()
    torch.cuda.synchronize()
    for ctxs in ([700, 300], [20, 299], [1, 0]):
        ins["ctx"].copy_(ints(ctxs))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        check(dict(x, ctxs=ctxs), out)
        assert torch.equal(out, second)
    assert ins["err"].item() == 0


# ---------------------------------------------------------------- acceptance
def drafts(r, lens, agree=0.7, padding=0):
    tokens, parents, choices = [], [], []
    for n in lens:
        p = make_tree(r, n, min(padding, n))
        c = r.randint(0, 9, n).tolist()
        t = [c[p[i]] if p[i] >= 0 and r.uniform() < agree else int(r.randint(0, 9)) for i in range(n)]
        tokens, parents, choices = tokens + t, parents + p, choices + c
    return tokens, parents, choices


@pytest.mark.parametrize("longest", [1, 2, 6, 300])
@pytest.mark.parametrize("lens", [[1], [8, 0, 30, 63], [256, 17], [3] * 70])
def test_accept_drafts(lens, longest):
    from cellm_b200 import ops
    r = np.random.RandomState(len(lens) + longest)
    tokens, parents, choices = drafts(r, lens, 0.9)
    e = err_word()
    count, path, after = ops.accept_drafts(ints(tokens), ints(parents), ints(choices), ints(np.concatenate([[0], np.cumsum(lens)])), longest, e)
    at = 0
    for b, n in enumerate(lens):
        want, token = plain.accept(tokens[at:at + n], parents[at:at + n], choices[at:at + n], longest)
        assert count[b].item() == len(want) and path[b].tolist() == want + [-1] * (longest - len(want)) and after[b].item() == token
        at += n
    assert e.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("items,nkv,hd,vd,page", [(3, 2, 64, 64, 16), (1, 1, 17, 17, 3), (2, 3, 10, 6, 5), (4, 1, 576, 0, 16), (16, 8, 64, 64, 16)])
def test_accepted_rows_go_into_the_pages(dtype, items, nkv, hd, vd, page):
    from cellm_b200 import ops
    r = np.random.RandomState(hd + page)
    lens, ctxs = [9, 1, 0, 40], [0, 7, 3, 61]
    tokens, parents, choices = drafts(r, lens, 0.95)
    T = sum(lens)
    table = r.permutation(4 * 40).reshape(4, 40)
    rows = {"k": torch.randn(T, items, nkv * hd + 2, device=DEV).to(dtype), "v": torch.randn(T, items, nkv * max(vd, 1) + 2, device=DEV).to(dtype)}
    sizes = {"k": hd, "v": vd}
    # a view whose nodes and items lie apart
    new = {x: rows[x][:, :, :nkv * sizes[x]].unflatten(2, (nkv, sizes[x])).transpose(0, 1) if sizes[x] else None for x in "kv"}
    pool = {x: torch.randn(items, 4 * 40, nkv, page, sizes[x], device=DEV).to(dtype) if sizes[x] else None for x in "kv"}
    want = {x: pool[x].clone() if sizes[x] else None for x in "kv"}
    e = err_word()
    count, path, _ = ops.accept_drafts(ints(tokens), ints(parents), ints(choices), ints(np.concatenate([[0], np.cumsum(lens)])), 12, e, k_new=new["k"],
                                       v_new=new["v"], k_pool=pool["k"], v_pool=pool["v"], ctx_lens=ints(ctxs), block_table=ints(table))
    at = 0
    for b, n in enumerate(lens):
        kept, _ = plain.accept(tokens[at:at + n], parents[at:at + n], choices[at:at + n], 12)
        for x in "kv":
            for j, i in enumerate(kept if sizes[x] else []):
                p = ctxs[b] + j
                want[x][:, table[b, p // page], :, p % page] = new[x][:, at + i]
        assert path[b].tolist()[:len(kept)] == kept
        at += n
    assert e.item() == 0 and all(torch.equal(pool[x], want[x]) for x in "kv" if sizes[x])


def test_trees_without_nodes_keep_nothing():
    from cellm_b200 import ops
    e, none, pool = err_word(), ints([]), torch.zeros(1, 4, 1, 2, 8, device=DEV)
    for more in ({}, dict(k_new=pool.new_zeros(1, 0, 1, 8), k_pool=pool, ctx_lens=ints([0, 3]), block_table=ints([[0, 1], [2, 3]]))):
        count, path, after = ops.accept_drafts(none, none, none, ints([0, 0, 0]), 3, e, **more)
        assert count.tolist() == [0, 0] and path.tolist() == [[-1] * 3] * 2 and after.tolist() == [-1, -1]
    count, path, after = ops.accept_drafts(none, none, none, ints([0]), 3, e)
    assert count.shape == after.shape == (0,) and path.shape == (0, 3) and e.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,ctx", [(33, 4000), (65, 9000), (64, 9000)])
def test_one_node_behind_a_long_context(dtype, hd, ctx):
    """One row whose keys are cut into an odd number of pieces, more than a cluster has."""
    x = make(np.random.RandomState(hd), dtype, [1], [ctx], 1, 1, hd, 16)
    check(x, run(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,nodes,nh,nkv", [(40, 3, 3, 1), (72, 5, 1, 1), (33, 1, 5, 1), (96, 7, 3, 3), (200, 3, 1, 1), (64, 1, 3, 1)])
@pytest.mark.parametrize("ctx", [130, 300, 517])
def test_pieces_of_a_cluster_share_rows_unevenly(dtype, hd, nodes, nh, nkv, ctx):
    """Two to eight pieces that merge in a cluster, each a share of the rows that is one row longer for one half of a warp than for the
    other, rows whose last columns only some lanes hold."""
    x = make(np.random.RandomState(hd + ctx), dtype, [nodes, nodes], [ctx, ctx - 70], nh, nkv, hd, 16)
    out = run(x)
    check(x, out)
    assert torch.equal(run(x), out)


def test_one_row_for_all_nodes():
    """Rows that are one row in memory (expanded), for few nodes and for as many as tiles of 128 rows are filled with."""
    r = np.random.RandomState(8)
    for n in (5, 40):
        x = make(r, torch.bfloat16, [n], [70], 8, 2, 64, 16)
        for name in ("q", "k_new", "v_new"):
            x[name] = x[name][:1].expand(n, -1)
        check(x, run(x))


def test_an_empty_cache():
    """Trees of requests without a committed token, over a pool without pages."""
    r = np.random.RandomState(4)
    for n in (5, 40):
        x = make(r, torch.bfloat16, [n], [0], 4, 2, 64, 16)
        check(x, run(x))
        check(x, run(dict(x, k=x["k"][:0], v=x["v"][:0], table=np.zeros((1, 0)))))


def test_acceptance_of_bad_trees_and_pages():
    from cellm_b200 import ops
    e = err_word()
    count, path, after = ops.accept_drafts(ints([5, 5, 5, 1]), ints([-1, 0, 3, -2]), ints([5, 5, 5, 5]), ints([0, 3, 4]), 3, e)
    assert e.item() == 32 and count.tolist() == [2, 0] and path.tolist() == [[0, 1, -1], [-1, -1, -1]] and after.tolist() == [5, -1]
    pool, new = torch.zeros(1, 4, 1, 2, 8, device=DEV), torch.ones(1, 3, 1, 8, device=DEV)
    for table, touched in ([[3, -1]], 2), ([[3, 4]], 2), ([[3]], 2):
        e, pool[:] = err_word(), 0.0
        count, _, _ = ops.accept_drafts(ints([5, 5, 5]), ints([-1, 0, 1]), ints([5, 5, 5]), ints([0, 3]), 4, e, k_new=new, k_pool=pool, ctx_lens=ints([0]), block_table=ints(table))
        assert e.item() == 2 and count.tolist() == [3] and pool.sum().item() == 8 * touched and pool[0, 3].sum().item() == 8 * touched


def test_a_step_of_drafting():
    """Trees of drafts through two layers as a program runs them: attention over the cache, the model's choices, acceptance; then the
    kept tokens are the request's context for the framework's own attention, which sees what the tree's nodes saw."""
    from cellm_b200 import ops
    r = np.random.RandomState(11)
    nh, nkv, hd, page, layers = 8, 2, 64, 16, 2
    lens, ctxs = [8, 21, 5], [30, 4, 129]
    T, B = sum(lens), len(lens)
    x = [make(np.random.RandomState(20 + i), torch.bfloat16, lens, ctxs, nh, nkv, hd, page, spare=4) for i in range(layers)]
    table = x[0]["table"]
    k_pool, v_pool = (torch.stack([y[z].nan_to_num(0.0) for y in x]) for z in "kv")
    k_new, v_new = (torch.stack([y[z].unflatten(1, (nkv, hd)) for y in x]) for z in ("k_new", "v_new"))
    tokens, parents, choices = drafts(r, lens, 0.95)
    e, cu = err_word(), ints(np.concatenate([[0], np.cumsum(lens)]))
    outs = [ops.attention_tree(x[i]["q"], k_new[i], v_new[i], ints(parents), k_pool[i], v_pool[i], cu, ints(ctxs), ints(table), lens, nh, hd ** -0.5, 0, e)
            for i in range(layers)]
    count, path, after = ops.accept_drafts(ints(tokens), ints(parents), ints(choices), cu, 8, e, k_new=k_new, v_new=v_new, k_pool=k_pool, v_pool=v_pool,
                                           ctx_lens=ints(ctxs), block_table=ints(table))
    assert e.item() == 0 and max(count.tolist()) > 1
    # every kept node, as a plain token at its place
    rows = [(b, j, sum(lens[:b]) + path[b, j].item()) for b in range(B) for j in range(count[b].item())]
    pos = ints([ctxs[b] + j for b, j, _ in rows])
    for i in range(layers):
        q = x[i]["q"][[t for _, _, t in rows]].contiguous()
        want = ops.attention_plain(q, k_pool[i], v_pool[i], pos, ints([b for b, _, _ in rows]), ints(table), nh, hd ** -0.5, 0, e)
        got = outs[i][[t for _, _, t in rows]]
        # both round what they hold of the weights and their result: four half steps of the largest value they weigh
        assert float((got.float() - want.float()).abs().max()) <= 4 * 2.0 ** -8 * float(torch.max(v_pool.abs().max(), v_new.abs().max()))
    assert e.item() == 0


def test_refusals():
    from cellm_b200 import ops
    r = np.random.RandomState(12)
    x = make(r, torch.bfloat16, [9, 4], [30, 2], 4, 2, 64, 16)
    good = dict(q=x["q"], k_new=x["k_new"], v_new=x["v_new"], parents=ints(x["parents"]), k_pool=x["k"], v_pool=x["v"], cu_seqlens=x["cu"], ctx_lens=ints(x["ctxs"]),
                block_table=ints(x["table"]), tree_lens=x["lens"], nh=4, scale=0.125, window=0, err=err_word())
    ops.attention_tree(**good)
    for bad in (dict(q=x["q"].float()), dict(q=x["q"][:, 1:]), dict(k_new=x["k_new"][:5]), dict(v_new=x["v_new"].cpu()), dict(k_new=x["k_new"].t().contiguous().t()),
                dict(parents=ints(x["parents"]).long()), dict(parents=ints(x["parents"])[:5]), dict(k_pool=x["k"][:, :1]), dict(v_pool=x["v"][:2]), dict(v_pool=x["v"].float()),
                dict(k_pool=x["k"].transpose(0, 1)), dict(cu_seqlens=x["cu"][:2]), dict(ctx_lens=ints([1])), dict(block_table=ints(x["table"])[:1]),
                dict(block_table=ints(x["table"]).t()), dict(tree_lens=[9, 5]), dict(tree_lens=[257, 4]), dict(tree_lens=[9]), dict(tree_lens=[9, -1]), dict(nh=3), dict(nh=0),
                dict(window=-1), dict(max_ctx=-1), dict(err=torch.zeros(1, device=DEV)), dict(err=torch.zeros(0, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            ops.attention_tree(**dict(good, **bad))
    new, pool = torch.zeros(2, 13, 2, 64, device=DEV), torch.zeros(2, 6, 2, 16, 64, device=DEV)
    good = dict(tokens=ints(x["parents"]), parents=ints(x["parents"]), choices=ints(x["parents"]), cu_seqlens=x["cu"], longest=3, err=err_word(), k_new=new, v_new=new,
                k_pool=pool, v_pool=pool.clone(), ctx_lens=ints([0, 0]), block_table=ints([[0, 1], [2, 3]]))
    ops.accept_drafts(**good)
    for bad in (dict(longest=0), dict(tokens=ints([1])), dict(choices=ints(x["parents"]).long()), dict(k_new=None), dict(k_pool=None), dict(v_pool=None), dict(ctx_lens=None),
                dict(ctx_lens=ints([0])), dict(block_table=None), dict(block_table=ints([[0]])), dict(k_new=new[:1]), dict(k_new=new.bfloat16()), dict(v_new=new[..., :32]),
                dict(v_pool=pool[:, :3]), dict(k_pool=pool.transpose(1, 2)), dict(k_new=new.transpose(2, 3).contiguous().transpose(2, 3)), dict(k_new=None, k_pool=None)):
        with pytest.raises(ValueError):
            ops.accept_drafts(**dict(good, **bad))
