"""Plain restatements, in 64 bits and one request after the other, of the operators that carry several continuations of a request:
attention of drafted trees, the acceptance of drafts, beam selection, and the reordering of states and cached rows."""
import math

import torch

F64 = torch.float64


def lineage(parents, i):
    """Node i and its ancestors, nearest first; None for padding and for what hangs on it."""
    line = []
    while i >= 0:
        line.append(i)
        i = parents[i]
    return line if i == -1 else None


def cached_rows(pool, entries, count):
    """[count, heads, size]: rows 0 .. count - 1 of a request whose pages are `entries`, from a pool [pages, heads, page size, size]."""
    ps = pool.shape[2]
    rows = [pool[entries[j // ps], :, j % ps] for j in range(count)]
    return torch.stack(rows) if rows else pool.new_zeros((0, pool.shape[1], pool.shape[3]))


def attention_tree(q, k_new, v_new, parents, k_pool, v_pool, lens, ctxs, table, nh, scale, window):
    """(outputs, sums of w |v|, bound of |scale q.k| formed by magnitudes, keys seen), each [T, nh, hd] or [T, nh]."""
    nkv, hd = k_pool.shape[1], k_pool.shape[3]
    T = sum(lens)
    out, mass = torch.zeros(T, nh, hd, dtype=F64), torch.zeros(T, nh, hd, dtype=F64)
    size, count = torch.zeros(T, nh, dtype=F64), torch.zeros(T, nh, dtype=F64)
    q, k_new, v_new = (x.to(F64).cpu().reshape(x.shape[0], -1, hd) for x in (q, k_new, v_new))
    base = 0
    for b, (n, ctx) in enumerate(zip(lens, ctxs)):
        k, v = (torch.cat([cached_rows(p.cpu(), table[b], ctx).to(F64), x[base:base + n]]) for p, x in ((k_pool, k_new), (v_pool, v_new)))
        for i in range(n):
            line = lineage(parents[base:base + n], i)
            if line is None:
                continue
            pos = ctx + len(line) - 1
            lo = max(0, pos - window + 1) if window else 0
            keys = list(range(lo, ctx)) + [ctx + a for a in (line[:window] if window else line)]
            for h in range(nh):
                z = scale * (k[keys, h // (nh // nkv)] @ q[base + i, h])
                w = torch.softmax(z, 0)
                out[base + i, h] = w @ v[keys, h // (nh // nkv)]
                mass[base + i, h] = w @ v[keys, h // (nh // nkv)].abs()
                size[base + i, h] = abs(scale) * (k[keys, h // (nh // nkv)].abs() @ q[base + i, h].abs()).max()
                count[base + i, h] = len(keys)
        base += n
    return out, mass, size, count


def accept(tokens, parents, choices, longest):
    """The places of one tree's standing nodes, and the token after them."""
    if not parents or parents[0] != -1:
        return [], -1
    path = [0]
    while len(path) < longest:
        fits = [i for i in range(len(parents)) if parents[i] == path[-1] and tokens[i] == choices[path[-1]]]
        if not fits:
            break
        path.append(fits[0])
    return path, choices[path[-1]]


def beams(logits, scores, keep, done, pad):
    """The sorted continuations [(score, beam, token)] of one request, and one more than `keep` of them."""
    found = []
    for k in range(len(scores)):
        s = float(scores[k])
        if s == -math.inf or math.isnan(s):
            continue
        if done is not None and bool(done[k]):
            found.append((s, k, pad))
            continue
        x = logits[k].to(F64).clone()
        x[torch.isnan(x)] = -math.inf
        z = torch.log_softmax(x, 0)
        found += [(s + float(z[v]), k, v) for v in torch.argsort(x, descending=True, stable=True)[:keep + 1].tolist() if float(x[v]) > -math.inf]
    return sorted(found, key=lambda f: (-f[0], f[1], f[2]))[:keep + 1]
