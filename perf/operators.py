"""The operators that carry several continuations of a request, as cases that can be timed and checked: trees of drafted
tokens and beams.

kinds:
  tree      attention of drafted trees over the paged cache (ops.attention_tree)
  accept    which drafted tokens stand, and their keys and values into the pages of every layer (ops.accept_drafts)
  beam      the best continuations of a request's beams (ops.beam_select)
  states    the beams' recurrent states in their new order (ops.reorder_states)
  pages     the beams' cached keys and values in their new order (ops.reorder_pages)

Each has a plain form in elementary torch operations beside the framework's call. Sizes are those of the shapes in
cellm_b200/config/presets.py ("1.2b": 32 heads over 8 of 64, 6 attention layers, vocabulary 65,536; "700m": 24 heads over 8),
pages of 16 tokens as the engine's.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
F64 = torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one user's request with a small tree behind a short prompt: the smallest call, bound by latency
        dict(name="tree 1x8", kind="tree", dtype="bfloat16", trees=1, nodes=8, context=500, ragged=False, heads=32, kv_heads=8, dim=64, page=16, window=0, padding=0),
        # a batch of requests that draft at once, contexts of all lengths
        dict(name="tree 16x25", kind="tree", dtype="bfloat16", trees=16, nodes=25, context=4096, ragged=True, heads=32, kv_heads=8, dim=64, page=16, window=0, padding=0),
        # large trees behind long documents: a tree's rows fill whole tiles of the tensor cores
        dict(name="tree 8x63 at 32768", kind="tree", dtype="bfloat16", trees=8, nodes=63, context=32768, ragged=False, heads=32, kv_heads=8, dim=64, page=16, window=0, padding=0),
        # the true 32-bit path, a window, groups of three heads, trees that were padded to one size
        dict(name="tree float32 window", kind="tree", dtype="float32", trees=5, nodes=13, context=3000, ragged=True, heads=24, kv_heads=8, dim=64, page=16, window=1024, padding=3),
        # the end of a single user's step: a walk down a small tree and a few rows of six layers
        dict(name="accept 1x8", kind="accept", dtype="bfloat16", trees=1, nodes=8, context=500, layers=6, kv_heads=8, dim=64, page=16, longest=6),
        # a full batch with large trees, sixteen attention layers
        dict(name="accept 64x63", kind="accept", dtype="bfloat16", trees=64, nodes=63, context=600, layers=16, kv_heads=8, dim=64, page=16, longest=16),
        # one user's four beams, one of them finished; an odd vocabulary in 16 bits
        dict(name="beam 1x4 bf16", kind="beam", dtype="bfloat16", requests=1, beams=4, keep=8, vocab=50257, done=1),
        # a batch of 64 requests with eight beams each
        dict(name="beam 64x8", kind="beam", dtype="float32", requests=64, beams=8, keep=16, vocab=65536, done=0),
        # the short convolutions' states of one user's beams
        dict(name="states 1x4 conv", kind="states", dtype="float32", requests=1, beams=4, layers=10, width=4096, slots=8),
        # matrix states (16 heads of 128 x 128) of a batch of beams
        dict(name="states 8x8 matrix", kind="states", dtype="float32", requests=8, beams=8, layers=10, width=262144, slots=64),
        # what one user's beams have generated so far
        dict(name="pages 1x4", kind="pages", dtype="bfloat16", requests=1, beams=4, prompt=300, rows=40, ragged=False, layers=6, kv_heads=8, dim=64, page=16),
        # a batch of beams with long answers
        dict(name="pages 16x8", kind="pages", dtype="bfloat16", requests=16, beams=8, prompt=500, rows=512, ragged=True, layers=6, kv_heads=8, dim=64, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    largest = {c["kind"]: work(c) for c in listed()}          # the last listed one of a kind that is not the smallest is its largest,
    largest["tree"] = work(listed()[2])                       # but for the trees
    while True:
        kind = rng.choice(["tree", "tree", "accept", "beam", "states", "pages"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        page = rng.choice([8, 16, 16, 32, 64])
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        dim = rng.choice([32, 64, 64, 64, 96, 128])
        if kind == "tree":
            c = dict(kind=kind, dtype=dtype, trees=_log(rng, 1, 64), nodes=_log(rng, 1, 128), context=_log(rng, 1, 32768), ragged=rng.random() < 0.7,
                     heads=kv_heads * rng.choice([1, 2, 3, 4, 4, 8]), kv_heads=kv_heads, dim=dim, page=page,
                     window=rng.choice([0, 0, _log(rng, 4, 2048)]), padding=0)
            c["padding"] = rng.choice([0, 0, rng.randint(0, c["nodes"] // 2)])
        elif kind == "accept":
            c = dict(kind=kind, dtype=dtype, trees=_log(rng, 1, 64), nodes=_log(rng, 1, 128), context=_log(rng, 1, 2000), layers=rng.randint(1, 16),
                     kv_heads=kv_heads, dim=dim, page=page, longest=rng.randint(1, 16))
        elif kind == "beam":
            beams = rng.randint(1, 16)
            c = dict(kind=kind, dtype=dtype, requests=_log(rng, 1, 64), beams=beams, keep=beams * rng.choice([1, 2, 2]), vocab=_log(rng, 1000, 150000),
                     done=rng.randint(0, beams - 1))
        elif kind == "states":
            c = dict(kind=kind, dtype=dtype, requests=_log(rng, 1, 32), beams=rng.randint(2, 16), layers=rng.randint(1, 16), width=_log(rng, 100, 262144), slots=0)
            c["slots"] = c["requests"] * c["beams"] + rng.randint(0, 8)
        else:
            c = dict(kind=kind, dtype=dtype, requests=_log(rng, 1, 32), beams=rng.randint(2, 16), prompt=_log(rng, 1, 1000), rows=_log(rng, 1, 1000),
                     ragged=rng.random() < 0.5, layers=rng.randint(1, 16), kv_heads=kv_heads, dim=dim, page=page)
        w = work(c)
        # 32-bit attention runs on a tenth of the bfloat16 rate, so it gets a tenth of the largest case's products
        if w["bytes"] <= largest[kind]["bytes"] and w["flops"] * (10 if c["kind"] == "tree" and c["dtype"] == "float32" else 1) <= max(largest[kind]["flops"], 1):
            return c


# ---------------------------------------------------------------- inputs
def _rng(seed):
    return np.random.RandomState(seed % (1 << 31))


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32 if math.prod(shape) < 1 << 26 else dtype).mul_(scale).to(dtype)


def _ints(values):
    return torch.as_tensor(np.asarray(values), dtype=torch.int32, device=DEV)


def _contexts(case):
    """Committed tokens of each tree's request: all `context`, or anything from none up to it."""
    r = np.random.RandomState(case["trees"] * 1009 + case["context"])
    return [int(x) for x in (r.uniform(0, 1, case["trees"]) ** 0.5 * case["context"])] if case["ragged"] else [case["context"]] * case["trees"]


def _spans(case):
    """How many rows each request's beams have generated, and behind how long a prompt."""
    r = np.random.RandomState(case["requests"] * 1013 + case["rows"])
    spread = lambda most: r.randint(max(1, most // 2), most + 1, case["requests"]) if case["ragged"] else np.full(case["requests"], most)  # noqa: E731
    return spread(case["rows"]), spread(case["prompt"])


def _tree(r, n, padding):
    """A drafted tree of n nodes, the last `padding` of them padding: a node hangs on one of the earlier ones, more often on a
    late one; now and then on the context itself, beside the first."""
    back = np.floor(r.uniform(0, 1, n) ** 2 * np.minimum(np.arange(n), 12)).astype(np.int64)
    parents = np.arange(n) - 1 - back
    parents[(np.arange(n) > 0) & (r.uniform(0, 1, n) < 0.04)] = -1
    parents[0] = -1
    parents[n - padding:] = -2
    if padding >= n:
        parents[0] = -1
    return parents


def _pages(r, lens, page):
    """Block tables of requests that hold `lens` tokens, on pages in no order, and the number of pages of the pool."""
    need = [-(-max(n, 1) // page) for n in lens]
    order = r.permutation(sum(need) + 3)
    table = np.full((len(lens), max(need)), -1)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order)


def prepare(case, seed):
    r, g = _rng(seed), _gen(seed)
    dt = TYPES[case["dtype"]]
    s = {"case": case, "err": torch.zeros(1, dtype=torch.int32, device=DEV)}
    kind = case["kind"]
    if kind in ("tree", "accept"):
        B, n, page, nkv, hd = case["trees"], case["nodes"], case["page"], case["kv_heads"], case["dim"]
        pad = case.get("padding", 0)
        parents = np.concatenate([_tree(r, n, pad) for _ in range(B)])
        ctx = _contexts(case) if kind == "tree" else [case["context"]] * B
        table, pages = _pages(r, [c + (n if kind == "accept" else 0) for c in ctx], page)
        s |= {"lens": [n] * B, "cu": _ints(np.arange(B + 1) * n), "ctx": _ints(ctx), "ctx_host": ctx, "table": _ints(table), "parents": _ints(parents)}
        if kind == "tree":
            # queries and the nodes' keys and values are columns of one product's rows, as a layer has them
            rows = _randn(g, B * n, (case["heads"] + 2 * nkv) * hd, dtype=dt)
            q_cols = case["heads"] * hd
            s |= {"q": rows[:, :q_cols].mul_(1.5), "k_new": rows[:, q_cols:q_cols + nkv * hd].unflatten(1, (nkv, hd)), "v_new": rows[:, q_cols + nkv * hd:].unflatten(1, (nkv, hd)),
                  "k": _randn(g, pages, nkv, page, hd, dtype=dt), "v": _randn(g, pages, nkv, page, hd, dtype=dt)}
        else:
            tokens = r.randint(0, 65536, B * n)
            choices = r.randint(0, 65536, B * n)
            first = np.repeat(np.arange(B) * n, n)
            hit = (r.uniform(0, 1, B * n) < 0.6) & (parents >= 0)
            tokens[hit] = choices[(first + np.maximum(parents, 0))[hit]]
            s |= {"tokens": _ints(tokens), "choices": _ints(choices)}
            for name in ("k", "v"):
                s[name] = _randn(g, case["layers"], pages, nkv, page, hd, dtype=dt)
                s[name + "_new"] = _randn(g, case["layers"], B * n, nkv, hd, dtype=dt)
    elif kind == "beam":
        R, K, V = case["requests"], case["beams"], case["vocab"]
        logits = _randn(g, R * K, V, dtype=torch.float32)
        logits += 4.0 * (torch.rand(R * K, V, generator=g, device=DEV) ** 12) * _randn(g, R * K, V).abs_()      # a few words are far likelier
        done = np.zeros((R, K), dtype=bool)
        done[:, K - case["done"]:] = r.uniform(0, 1, (R, case["done"])) < 0.7
        s |= {"logits": logits.to(dt), "scores": (-torch.rand(R, K, generator=g, device=DEV) * 3 - 20.0),
              "done": torch.as_tensor(done, device=DEV) if case["done"] else None}
    else:
        R, K = case["requests"], case["beams"]
        # the next best continuations come from about two thirds of the beams; most change their place
        parents = r.randint(0, K, (R, K)) * (r.uniform(0, 1, (R, K)) < 0.9) + 0
        s["parents"] = _ints(parents)
        if kind == "states":
            s |= {"state": _randn(g, case["layers"], case["slots"], case["width"], dtype=dt), "slots": _ints(r.permutation(case["slots"])[:R * K])}
        else:
            lens, starts = _spans(case)
            ends = starts + lens
            table, pages = _pages(r, np.repeat(ends, K).tolist(), case["page"])
            shape = (case["layers"], pages, case["kv_heads"], case["page"], case["dim"])
            s |= {"starts": _ints(starts), "ends": _ints(ends), "table": _ints(table), "longest": int(lens.max()),
                  "k": _randn(g, *shape, dtype=dt), "v": _randn(g, *shape, dtype=dt)}
    return s


# ---------------------------------------------------------------- plain forms
def _lineage(parents, cu, n):
    """[B, n, n]: whether node j is node i or one of its ancestors; padding nodes have none."""
    p = parents.view(-1, n).long()
    up = (p.unsqueeze(2) == torch.arange(n, device=p.device)).to(F64)
    line = torch.linalg.matrix_power(up + torch.eye(n, device=p.device, dtype=F64), max(n - 1, 1)) > 0
    return line & (p >= -1).unsqueeze(2)


def _plain_tree(s):
    c = s["case"]
    B, n, nh, nkv, hd, ps, window = c["trees"], c["nodes"], c["heads"], c["kv_heads"], c["dim"], c["page"], c["window"]
    G, L = nh // nkv, max(s["ctx_host"])
    line = _lineage(s["parents"], s["cu"], n)
    depth = line.sum(2) - 1
    j = torch.arange(L, device=DEV)
    page = s["table"].long()[:, j // ps].clamp(min=0)
    k = torch.cat([s["k"][page, :, j % ps].float(), s["k_new"].view(B, n, nkv, hd).float()], 1)
    v = torch.cat([s["v"][page, :, j % ps].float(), s["v_new"].view(B, n, nkv, hd).float()], 1)
    ctx = s["ctx"].long().view(B, 1, 1)
    first = ctx + depth.unsqueeze(2) - window + 1 if window else torch.zeros_like(ctx)
    sees = torch.cat([((j < ctx) & (j >= first)).expand(B, n, L), line & (depth.unsqueeze(2) - depth.unsqueeze(1) < window) if window else line], 2)
    sees &= line.any(2, keepdim=True)                                                                    # [B, n, L + n]
    q = s["q"].reshape(B, n, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * n, hd).float()
    z = (q @ k.permute(0, 2, 3, 1)).mul_(hd ** -0.5).view(B, nkv, G, n, L + n)
    z.masked_fill_(~sees.view(B, 1, 1, n, L + n), -math.inf)
    top = z.amax(-1, keepdim=True)
    e = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(B, nkv, G * n, L + n) @ v.permute(0, 2, 1, 3)).view(B, nkv, G, n, hd) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(B * n, nh * hd).to(s["q"].dtype)


def _plain_accept(s):
    c = s["case"]
    B, n, ps = c["trees"], c["nodes"], c["page"]
    line = _lineage(s["parents"], s["cu"], n)
    p, tokens, choices = s["parents"].view(B, n).long(), s["tokens"].view(B, n), s["choices"].view(B, n)
    fits = (p >= 0) & (tokens == choices.gather(1, p.clamp(min=0)))
    i = torch.arange(n, device=DEV)
    earlier = (p.unsqueeze(2) == p.unsqueeze(1)) & fits.unsqueeze(1) & (i.view(n, 1) > i)                # an earlier sibling fits too
    fits &= ~earlier.any(2)
    fits[:, 0] = True
    depth = line.sum(2) - 1
    stands = ~(line & ~fits.unsqueeze(1)).any(2) & (p >= -1) & (depth < c["longest"])
    count = stands.sum(1)
    path = torch.full((B, c["longest"] + 1), -1, dtype=torch.int64, device=DEV)
    path.scatter_(1, torch.where(stands, depth, c["longest"]), torch.where(stands, i, -1))
    path = path[:, :c["longest"]]
    after = choices.gather(1, path.gather(1, (count - 1).unsqueeze(1))).squeeze(1)
    place = (s["ctx"].long().view(B, 1) + depth)[stands]
    b = torch.arange(B, device=DEV).view(B, 1).expand(B, n)[stands]
    page, row = s["table"].long()[b, place // ps], (torch.arange(B * n, device=DEV).view(B, n))[stands]
    for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        pool[:, page, :, place % ps] = new[:, row].transpose(0, 1)
    return count.int(), path.int(), after.int(), s["k"], s["v"]


def _plain_beam(s):
    c = s["case"]
    R, K, V = c["requests"], c["beams"], c["vocab"]
    x = s["logits"].to(F64).view(R, K, V)
    top = x.amax(-1, keepdim=True)
    z = s["scores"].to(F64).unsqueeze(2) + (x - ((x - top).exp_().sum(-1, keepdim=True).log_() + top))
    if s["done"] is not None:
        alone = torch.full_like(z, -math.inf)
        alone[:, :, 0] = s["scores"].to(F64)
        z = torch.where(s["done"].unsqueeze(2), alone, z)
    score, at = z.view(R, K * V).sort(dim=1, descending=True, stable=True)
    score, at = score[:, :c["keep"]], at[:, :c["keep"]]
    fine = score > -math.inf
    return score.float(), torch.where(fine, at // V, -1).int(), torch.where(fine, at % V, -1).int()


def _plain_states(s):
    R, K = s["case"]["requests"], s["case"]["beams"]
    slots = s["slots"].long().view(R, K)
    s["state"][:, slots.view(-1)] = s["state"][:, slots.gather(1, s["parents"].long()).view(-1)]
    return s["state"]


def _plain_pages(s):
    c = s["case"]
    R, K, ps = c["requests"], c["beams"], c["page"]
    at = s["starts"].long().view(R, 1) + torch.arange(s["longest"], device=DEV)                            # [R, rows]
    moved = ((at < s["ends"].view(R, 1)).unsqueeze(1) & (s["parents"] != torch.arange(K, device=DEV)).unsqueeze(2))
    width = s["table"].shape[1]
    page = s["table"].long().view(R, K, width).gather(2, (at // ps).clamp(max=width - 1).unsqueeze(1).expand(R, K, -1))
    source = page.gather(1, s["parents"].long().unsqueeze(2).expand_as(page))
    slot = (at % ps).unsqueeze(1).expand_as(page)[moved]
    for pool in (s["k"], s["v"]):
        pool[:, page[moved], :, slot] = pool[:, source[moved], :, slot]
    return s["k"], s["v"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return {"tree": _plain_tree, "accept": _plain_accept, "beam": _plain_beam, "states": _plain_states, "pages": _plain_pages}[kind](s)
    from cellm_b200 import ops
    if kind == "tree":
        return ops.attention_tree(s["q"], s["k_new"], s["v_new"], s["parents"], s["k"], s["v"], s["cu"], s["ctx"], s["table"], s["lens"], c["heads"],
                                  c["dim"] ** -0.5, c["window"], s["err"], max_ctx=max(s["ctx_host"]))
    if kind == "accept":
        count, path, after = ops.accept_drafts(s["tokens"], s["parents"], s["choices"], s["cu"], c["longest"], s["err"], k_new=s["k_new"], v_new=s["v_new"],
                                               k_pool=s["k"], v_pool=s["v"], ctx_lens=s["ctx"], block_table=s["table"])
        return count, path, after, s["k"], s["v"]
    if kind == "beam":
        return ops.beam_select(s["logits"], s["scores"], c["keep"], done=s["done"])
    if kind == "states":
        ops.reorder_states(s["state"], s["slots"], s["parents"], s["err"])
        return s["state"]
    ops.reorder_pages(s["k"], s["v"], s["table"], s["starts"], s["ends"], s["parents"], s["err"])
    return s["k"], s["v"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, kind = case, case["kind"]
    e = 2 if c["dtype"] == "bfloat16" else 4
    if kind == "tree":
        B, n, nh, nkv, hd = c["trees"], c["nodes"] - c["padding"], c["heads"], c["kv_heads"], c["dim"]
        keys = sum(min(x, c["window"]) if c["window"] else x for x in _contexts(c))
        return {"bytes": (2 * keys * nkv + B * n * (2 * nh + 2 * nkv)) * hd * e, "flops": 4.0 * nh * hd * n * (keys + B * (n + 1) / 2)}
    if kind == "accept":
        # about one node in four of the longest path stands: its rows are read and written
        rows = c["trees"] * max(1, min(c["longest"], c["nodes"]) // 4)
        return {"bytes": 12 * c["trees"] * c["nodes"] + 4.0 * rows * c["layers"] * c["kv_heads"] * c["dim"] * e, "flops": 0}
    if kind == "beam":
        return {"bytes": c["requests"] * (c["beams"] * c["vocab"] * e + 8 * c["beams"] + 12 * c["keep"]), "flops": 4.0 * c["requests"] * c["beams"] * c["vocab"]}
    # of K beams that get K parents at random, 1 - 1/K move, and they come from about 1 - 1/e of the beams
    R, K = c["requests"], c["beams"]
    moved, sources = R * (K - 1), R * K * (1 - (1 - 1 / K) ** K)
    if kind == "states":
        return {"bytes": (moved + sources) * c["layers"] * c["width"] * e, "flops": 0}
    return {"bytes": 2.0 * (moved + sources) * float(np.mean(_spans(c)[0])) * c["layers"] * c["kv_heads"] * c["dim"] * e, "flops": 0}


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "beam": _exact_beam, "states": lambda s: None, "pages": lambda s: None}[case["kind"]](s)


def _ancestors(parents):
    """For each node of one tree the list of itself and its ancestors, nearest first; None for padding."""
    out = []
    for i, p in enumerate(parents):
        out.append(None if p < -1 else [i] + (out[p] if p >= 0 else []))
    return out


def _exact_tree(s):
    c = s["case"]
    n, nh, nkv, hd, ps, window = c["nodes"], c["heads"], c["kv_heads"], c["dim"], c["page"], c["window"]
    table, parents = s["table"].tolist(), s["parents"].tolist()
    out = torch.zeros(c["trees"] * n, nh, hd, dtype=F64, device=DEV)
    for b, ctx in enumerate(s["ctx_host"]):
        pages = torch.tensor(table[b][:-(-ctx // ps)], dtype=torch.long, device=DEV)
        rows = slice(b * n, (b + 1) * n)
        k, v = (torch.cat([s[x][pages].transpose(1, 2).reshape(-1, nkv, hd)[:ctx], s[x + "_new"][rows]]).to(F64) for x in ("k", "v"))
        sees = torch.zeros(n, ctx + n, dtype=torch.bool)
        for i, line in enumerate(_ancestors(parents[rows])):
            if line is not None:
                sees[i, max(0, ctx + len(line) - window) if window else 0:ctx] = True
                sees[i, [ctx + a for a in (line[:window] if window else line)]] = True
        sees = sees.to(DEV)
        for h in range(nh):
            z = s["q"][rows, h * hd:(h + 1) * hd].to(F64) @ k[:, h // (nh // nkv)].T / math.sqrt(hd)
            w = torch.softmax(z.masked_fill(~sees, -math.inf), 1).nan_to_num(0.0)
            out[rows, h] = w @ v[:, h // (nh // nkv)]
    return out.view(-1, nh * hd)


def _exact_accept(s):
    c = s["case"]
    n = c["nodes"]
    count, path, after = [], [], []
    for b in range(c["trees"]):
        tokens, parents, choices = (s[x].tolist()[b * n:(b + 1) * n] for x in ("tokens", "parents", "choices"))
        line = [0]
        while len(line) < c["longest"]:
            child = [i for i in range(n) if parents[i] == line[-1] and tokens[i] == choices[line[-1]]]
            if not child:
                break
            line.append(child[0])
        count.append(len(line))
        path.append(line + [-1] * (c["longest"] - len(line)))
        after.append(choices[line[-1]])
    return _ints(count), _ints(path), _ints(after), None, None


def _exact_beam(s):
    c = s["case"]
    R, K, V = c["requests"], c["beams"], c["vocab"]
    scores, parents, tokens = [], [], []
    for r in range(R):
        found = []
        for k in range(K):
            score = float(s["scores"][r, k])
            if s["done"] is not None and bool(s["done"][r, k]):
                found.append((-score, k, 0))
                continue
            x = torch.log_softmax(s["logits"][r * K + k].to(F64), 0)
            last = x.kthvalue(max(1, V - c["keep"] + 1)).values
            at = torch.nonzero(x >= last).view(-1)
            found += [(-(score + z), k, v) for z, v in zip(x[at].tolist(), at.tolist())]
        found = sorted(found)[:c["keep"]]
        found += [(math.inf, -1, -1)] * (c["keep"] - len(found))
        scores.append([-f[0] for f in found])
        parents.append([f[1] for f in found])
        tokens.append([f[2] for f in found])
    return torch.tensor(scores, dtype=F64, device=DEV), _ints(parents), _ints(tokens)
