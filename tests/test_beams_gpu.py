"""Beam selection and the reordering of beams' states and cached rows against plain 64-bit restatements: ties, finished beams, rows
without a choice, odd vocabularies, strided rows; states of any width, pages of any size, beams that share a parent or swap."""
import math

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


def check_selection(logits, scores, keep, done=None, pad=0):
    from cellm_b200 import ops
    R, K = scores.shape
    got_s, got_p, got_t = (x.cpu() for x in ops.beam_select(logits, scores, keep, done=done, pad=pad))
    lc, sc, dc = logits.cpu(), scores.cpu(), None if done is None else done.cpu()
    for r in range(R):
        want = plain.beams(lc[r * K:(r + 1) * K], sc[r], keep, None if dc is None else dc[r], pad)
        n = min(keep, len(want))
        picked = list(zip(got_p[r].tolist(), got_t[r].tolist()))
        assert picked[n:] == [(-1, -1)] * (keep - n) and got_s[r, n:].tolist() == [-math.inf] * (keep - n)
        assert len(set(picked[:n])) == n
        exact = {(k, v): s for s, k, v in want}
        for i in range(n):
            s, k, v = want[i]
            # a score is rounded once, and the sum behind it carries 2^-23 at most
            assert abs(float(got_s[r, i]) - s) <= 2.0 ** -24 * abs(s) + 2.0 ** -22
            # two beams' continuations nearer than what their sums carry may change places; all else stands where it belongs
            near = [w for w in want if abs(w[0] - s) <= 2.0 ** -21]
            if len({w[1] for w in near}) == 1 or all(w[0] == s for w in near):
                if i + 1 < len(want) or len(near) == 1:
                    assert picked[i] == (k, v), (r, i, picked[i], (k, v))
            else:
                assert picked[i] in exact


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,K,keep,V", [(1, 1, 1, 1), (1, 4, 8, 65536), (3, 5, 10, 50257), (2, 8, 16, 1000), (7, 2, 4, 131), (1, 32, 64, 2048), (2, 3, 64, 5), (5, 16, 32, 8193)])
def test_selection(dtype, R, K, keep, V):
    torch.manual_seed(V + K)
    logits = (torch.randn(R * K, V) * 3).to(dtype).to(DEV)
    check_selection(logits, -torch.rand(R, K, device=DEV) * 5, keep)
    first = torch.full((R, K), -math.inf, device=DEV)                    # the first step: one beam has a score
    first[:, 0] = 0.0
    check_selection(logits, first, keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [777, 50257])
def test_equal_logits_are_taken_by_beam_and_token(dtype, V):
    """Rows of few different values, of one value, of the type's lowest value, of -inf, with a NaN here and there, and very large ones."""
    torch.manual_seed(V)
    rows = [torch.randint(0, 3, (V,)).float(), torch.zeros(V), torch.full((V,), float(torch.finfo(dtype).min)), torch.full((V,), -math.inf),
            torch.randint(0, 2, (V,)).float() * 5, torch.randn(V), torch.full((V,), 3.0e6), torch.linspace(-50, 50, V)]
    rows[4][::5] = -math.inf
    rows[5][::7] = math.nan
    logits = torch.stack(rows).to(dtype).to(DEV)
    for keep in (1, 5, 64):
        check_selection(logits, torch.zeros(8, 1, device=DEV), keep)
        check_selection(logits, torch.tensor([[0.0, -1.0, -2.0, -3.0], [0.0, -30.0, -2.0, -1.5]], device=DEV), keep)
    check_selection(logits[:2].repeat(2, 1), torch.zeros(1, 4, device=DEV), 64)                    # beams that are alike


def test_finished_beams_offer_themselves():
    torch.manual_seed(2)
    logits = torch.randn(12, 3001, device=DEV)
    logits[3] = math.nan                                   # a finished beam's row is not looked at
    scores = torch.tensor([[-9.0, -3.0, -4.0, -2.0], [-9.0, -8.0, -4.0, -20.0], [-1.0, -math.inf, -2.0, -1.0]], device=DEV)
    done = torch.tensor([[False, False, True, True], [True, True, True, True], [True, True, False, True]], device=DEV)
    for keep in (2, 8):
        check_selection(logits, scores, keep, done, pad=7)


def test_rows_may_lie_apart_and_anywhere():
    torch.manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(6, 5003, device=DEV).to(dtype)
        scores = -torch.rand(2, 3, device=DEV)
        for lo, hi in ((0, 5000), (1, 4999), (3, 5003)):
            check_selection(wide[:, lo:hi], scores, 6)


# An exponential is off by 1.1e-7 of itself at most (its argument by two halves of 2^-25 units of log 2, the polynomial's last three
# roundings by 2^-24, 2^-26 and less, its fit by 3e-9), sums of eight by three half steps of 2^-23; what follows is 64 bits.
SUM_ERROR = 3.0e-7


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1024, 50257])
@pytest.mark.parametrize("flat,top", [(0.1, 8.35), (1.3, 8.8), (-5.2, 1.9), (-40000.0, -39990.5), (32760.0, 32770.0), (0.3, 0.7)])
def test_sums_of_flat_rows_with_an_outlier(dtype, V, flat, top):
    """A row's mass several units below its largest logit, of equal logits: their errors have one sign. The beams' scores are their rows'
    log-sums, so that what is left shows the error and not a score's own rounding."""
    from cellm_b200 import ops
    row = torch.full((V,), flat, dtype=dtype)
    row[::1024] = top
    exact = row.double()
    z = torch.logsumexp(exact, 0) - exact.max()
    start = z.float()
    got, _, tokens = ops.beam_select(row.to(DEV).unsqueeze(0), start.view(1, 1).to(DEV), 1)
    assert tokens.item() == 0 and abs(float(got) - float(start.double() - z)) <= SUM_ERROR


def left_of(row):
    """What beam_select leaves of a score that is the row's log-sum below its largest logit, against the same in 64 bits: the error of the
    kernels' log-sum."""
    from cellm_b200 import ops
    exact = row.double()
    z = torch.logsumexp(exact, 0) - exact.max()
    start = z.float()
    got, _, _ = ops.beam_select(row.to(DEV).unsqueeze(0), start.view(1, 1).to(DEV), 1)
    return abs(float(got) - float(start.double() - z))


def test_logarithms_of_sums():
    """Rows of zeros, whose exponentials and sums are exact: log V where log2 V lies halfway between whole numbers, the exponential's far
    end. Its fit is good to 2.0e-9, the 32-bit logarithm's error enters squared."""
    for V in (181, 362, 23170, 46341):
        assert left_of(torch.zeros(V)) <= 2.5e-9, V


def test_exponentials_of_a_narrow_range():
    """65,536 logits whose exponentials lie at the polynomial's far end. Single roundings (1.1e-7 at most) average out to less than 3e-9 of six
    deviations; the error of its fit (3.0e-9, and 2.0e-9 of the logarithm) does not, nor does the last rounding of its argument: x times
    log2 e's second part, 1.9e-8 x, is nearly the same for all of them and is added to a multiple of 2^-25, half a step of which is
    2^-26 log 2 = 1.03e-8 of an exponential. 1.84e-8 in all."""
    torch.manual_seed(5)
    for n in (0, 3, -7):
        row = ((n + 0.44 + 0.06 * torch.rand(65536, dtype=torch.float64)) * math.log(2)).float()
        assert left_of(row) <= 1.84e-8, n
        row = ((n - 0.5 + 0.06 * torch.rand(65536, dtype=torch.float64)) * math.log(2)).float()
        assert left_of(row) <= 1.84e-8, n


def test_exponentials_of_a_range_without_that_rounding():
    """The same between 3.0782 and 3.1192 in magnitude, whose log2 leave 0.441 to 0.4999 above or below whole numbers, and of which log2 e's
    second part makes 1.989 to 2.0155 steps of 2^-25: 5e-10 are lost. 8.5e-9 in all."""
    torch.manual_seed(6)
    for sign in (1, -1):
        assert left_of((sign * (3.0782 + 0.041 * torch.rand(65536, dtype=torch.float64))).float()) <= 8.5e-9, sign


def test_a_captured_selection_follows_its_inputs():
    from cellm_b200 import ops
    logits, scores = torch.randn(8, 9000, device=DEV), torch.zeros(2, 4, device=DEV)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.beam_select(logits, scores, 8)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = ops.beam_select(logits, scores, 8)
    for seed in range(3):
        torch.manual_seed(seed)
        logits.copy_(torch.randn(8, 9000))
        scores.copy_(-torch.rand(2, 4))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.beam_select(logits, scores, 8)))


def some_parents(r, R, K):
    parents = r.randint(0, K, (R, K))
    parents[0] = np.roll(np.arange(K), 1)                  # a ring: every beam takes its neighbour's
    if R > 1:
        parents[1] = K - 1                                 # all follow one
        parents[1, 0] = -1
    return parents


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("R,K,items,shape", [(1, 4, 10, (2, 2048)), (3, 5, 2, (7,)), (2, 1, 1, (64,)), (2, 32, 3, (9, 33)), (4, 16, 1, (16, 128)), (9, 2, 2, (1,)), (2, 9, 1, (40001,))])
def test_states_follow_their_beams(dtype, R, K, items, shape):
    from cellm_b200 import ops
    r = np.random.RandomState(R + K)
    slots = R * K + 3
    state = torch.randn(items, slots, *shape, device=DEV).to(dtype)
    at, parents = r.permutation(slots)[:R * K], some_parents(r, R, K)
    want = state.clone()
    for q in range(R):
        for k in range(K):
            if parents[q, k] >= 0:
                want[:, at[q * K + k]] = state[:, at[q * K + parents[q, k]]]
    e = err_word()
    ops.reorder_states(state, ints(at), ints(parents), e)
    assert torch.equal(state, want) and e.item() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [2, 4, 7, 13, 20])
@pytest.mark.parametrize("width", [2047, 2049, 4098, 5001, 70001])
def test_states_of_odd_widths(dtype, K, width):
    """Units of 2, 4 and 8 bytes, several of them a thread, and the last of a slot's among them."""
    from cellm_b200 import ops
    r = np.random.RandomState(width + K)
    state = torch.randn(2, 2 * K + 1, width, device=DEV).to(dtype)
    at, parents = r.permutation(2 * K + 1)[:2 * K], some_parents(r, 2, K)
    want = state.clone()
    for q in range(2):
        for k in range(K):
            if parents[q, k] >= 0:
                want[:, at[q * K + k]] = state[:, at[q * K + parents[q, k]]]
    e = err_word()
    ops.reorder_states(state, ints(at), ints(parents), e)
    assert torch.equal(state, want) and e.item() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,K,items,nkv,page,hd,vd", [(1, 4, 6, 8, 16, 64, 64), (3, 5, 1, 1, 3, 17, 17), (2, 32, 2, 2, 8, 32, 32), (2, 3, 2, 1, 16, 576, 0), (4, 9, 3, 2, 16, 96, 128)])
def test_cached_rows_follow_their_beams(dtype, R, K, items, nkv, page, hd, vd):
    from cellm_b200 import ops
    r = np.random.RandomState(R + K + page)
    ends = r.randint(1, 70, R)
    starts = np.array([r.randint(0, e + 1) for e in ends])
    starts[0], ends[-1] = 0, 70
    entries = -(-70 // page)
    table = r.permutation(R * K * entries).reshape(R * K, entries)
    parents = some_parents(r, R, K)
    given_back = (starts[-1] // page) if R > 1 else -1           # a page that every beam of a request has given back
    pools = [torch.randn(items, R * K * entries, nkv, page, d, device=DEV).to(dtype) for d in (hd, vd) if d]
    want = [p.clone() for p in pools]
    if given_back >= 0:
        table[(R - 1) * K:, given_back] = -1
    for q in range(R):
        for k in range(K):
            for at in range(starts[q], ends[q]):
                to, src = (table[q * K + x, at // page] for x in (k, parents[q, k]))
                if parents[q, k] >= 0 and to >= 0:
                    for w, p in zip(want, pools):
                        w[:, to, :, at % page] = p[:, src, :, at % page]
    e = err_word()
    ops.reorder_pages(pools[0], pools[1] if vd else None, ints(table), ints(starts), ints(ends), ints(parents), e)
    assert e.item() == 0 and all(torch.equal(p, w) for p, w in zip(pools, want))


@pytest.mark.parametrize("K", [2, 3, 4, 20])
@pytest.mark.parametrize("hd", [8, 4, 2])
def test_pages_of_many_rows(K, hd):
    """Enough rows that blocks look many of them up at a time; starts and ends inside and outside of such runs; units of 16, 8 and 4 bytes."""
    from cellm_b200 import ops
    r = np.random.RandomState(K + hd)
    R, items, nkv, page, entries = 6, 3, 2, 16, 50
    pool = torch.randn(items, R * K * entries, nkv, page, hd, device=DEV).to(torch.bfloat16)
    table, parents = r.permutation(R * K * entries).reshape(R * K, entries), some_parents(r, R, K)
    starts, ends = [0, 33, 500, 7, 64, 799], [800, 797, 501, 7, 96, 800]
    places = torch.from_numpy(table[:, np.arange(800) // page] * page + np.arange(800) % page).to(DEV)      # of every beam's rows, in a pool of single rows
    rows = pool.permute(0, 2, 1, 3, 4).reshape(items * nkv, -1, hd)
    want = rows.clone()
    for q in range(R):
        for k in range(K):
            if parents[q, k] >= 0:
                to, src = (places[q * K + x, starts[q]:ends[q]] for x in (k, int(parents[q, k])))
                want[:, to] = rows[:, src]
    e = err_word()
    ops.reorder_pages(pool, None, ints(table), ints(starts), ints(ends), ints(parents), e)
    assert e.item() == 0 and torch.equal(pool.permute(0, 2, 1, 3, 4).reshape(items * nkv, -1, hd), want)


def test_bad_parents_slots_and_pages_are_reported_and_passed_over():
    from cellm_b200 import ops
    state = torch.arange(5.0, device=DEV).repeat(2, 1).unsqueeze(2).contiguous()
    e = err_word()
    ops.reorder_states(state, ints([3, 1, 4]), ints([[1, 3, 0]]), e)
    assert e.item() == 4 and state[0].flatten().tolist() == [0, 1, 2, 1, 3]
    state = torch.arange(5.0, device=DEV).repeat(2, 1).unsqueeze(2).contiguous()
    e = err_word()
    ops.reorder_states(state, ints([3, 5, -1]), ints([[1, 0, 0]]), e)
    assert e.item() == 4 and state[0].flatten().tolist() == [0, 1, 2, 3, 4]
    pool = torch.arange(6.0, device=DEV).view(1, 6, 1, 1, 1).repeat(1, 1, 1, 2, 4).contiguous()
    e = err_word()
    ops.reorder_pages(pool, None, ints([[0, 1], [2, 6], [4, 5]]), ints([0]), ints([4]), ints([[1, 2, 2]]), e)
    assert e.item() == 2 and pool[0, :, 0, 0, 0].tolist() == [2, 1, 4, 3, 4, 5]
    pool = torch.arange(6.0, device=DEV).view(1, 6, 1, 1, 1).repeat(1, 1, 1, 2, 4).contiguous()
    e = err_word()
    ops.reorder_pages(pool, None, ints([[0, 1], [2, 3], [4, 5]]), ints([3]), ints([9]), ints([[1, 5, 0]]), e)
    assert e.item() == 2 | 4 and pool[0, :, 0].tolist()[1] == [[1.0] * 4, [3.0] * 4] and pool[0, :, 0].tolist()[5] == [[5.0] * 4, [1.0] * 4]


def test_negative_parents_pages_and_rows_are_reported_too():
    """-1 says that a beam stays and that a page was given back; anything below it, and a row before the first, is out of range: reported
    and passed over as the other end's."""
    from cellm_b200 import ops
    state = torch.arange(5.0, device=DEV).repeat(2, 1).unsqueeze(2).contiguous()
    for parent, said in ((-1, 0), (-2, 4), (-2 ** 31, 4)):
        e = err_word()
        ops.reorder_states(state, ints([3, 1, 4]), ints([[0, parent, 2]]), e)
        assert e.item() == said and state[0].flatten().tolist() == [0, 1, 2, 3, 4]
    base = torch.arange(6.0, device=DEV).view(1, 6, 1, 1, 1).repeat(1, 1, 1, 2, 4).contiguous()
    for table, start, parents, said, rows in (([[0, 1], [2, 3], [4, 5]], 0, [1, -2, 2], 4, [2, 3, 2, 3, 4, 5]), ([[0, 1], [2, -1], [4, 5]], 0, [0, 2, 2], 0, [0, 1, 4, 3, 4, 5]),
                                              ([[0, 1], [2, -2], [4, 5]], 0, [0, 2, 2], 2, [0, 1, 4, 3, 4, 5]), ([[0, 1], [2, 3], [4, 5]], -3, [2, 1, 2], 2, [4, 5, 2, 3, 4, 5])):
        pool, e = base.clone(), err_word()
        ops.reorder_pages(pool, None, ints(table), ints([start]), ints([4]), ints([parents]), e)
        assert e.item() == said and pool[0, :, 0, 0, 0].tolist() == rows and pool[0, :, 0, 1, 3].tolist() == rows


def test_a_search_through_its_steps():
    """Beams of two requests over a cache with states and pages, six steps: selection, then reordering, each beam writing its token into its
    state and its rows; at the end every beam's state and rows spell the tokens of its own history."""
    from cellm_b200 import ops
    R, K, V, steps, prompt, page = 2, 4, 500, 6, 5, 4
    torch.manual_seed(9)
    r = np.random.RandomState(9)
    state = torch.zeros(3, R * K + 1, steps, device=DEV)
    entries = -(-(prompt + steps) // page)
    table = r.permutation(R * K * entries).reshape(R * K, entries)
    pool = torch.zeros(2, R * K * entries, 1, page, 8, device=DEV)
    slots, e = r.permutation(R * K + 1)[:R * K], err_word()
    scores = torch.full((R, K), -math.inf, device=DEV)
    scores[:, 0] = 0.0
    histories = [[[] for _ in range(K)] for _ in range(R)]
    for step in range(steps):
        logits = torch.randn(R * K, V, device=DEV) * 2
        want = [plain.beams(logits[q * K:(q + 1) * K].cpu(), scores[q].cpu(), K, None, 0)[:K] for q in range(R)]
        scores, parents, tokens = ops.beam_select(logits, scores, K)
        assert [[(k, v) for _, k, v in w] for w in want] == [list(zip(p, t)) for p, t in zip(parents.tolist(), tokens.tolist())]
        ops.reorder_states(state, ints(slots), parents, e)
        ops.reorder_pages(pool, None, ints(table), ints([prompt] * R), ints([prompt + step] * R), parents, e)
        histories = [[histories[q][p] + [t] for p, t in zip(parents[q].tolist(), tokens[q].tolist())] for q in range(R)]
        at = prompt + step
        for q in range(R):
            for k in range(K):
                state[:, slots[q * K + k], step] = tokens[q, k].float()
                pool[:, table[q * K + k, at // page], :, at % page] = tokens[q, k].float()
    for q in range(R):
        for k in range(K):
            assert state[1, slots[q * K + k]].tolist() == histories[q][k]
            assert [pool[1, table[q * K + k, a // page], 0, a % page, 3].item() for a in range(prompt, prompt + steps)] == histories[q][k]
    assert e.item() == 0


def test_refusals():
    from cellm_b200 import ops
    logits, scores = torch.zeros(6, 50, device=DEV), torch.zeros(2, 3, device=DEV)
    for a, k in (((logits.half(), scores, 2), {}), ((logits, scores.double(), 2), {}), ((logits, scores.view(3, 2).t(), 2), {}), ((logits, torch.zeros(3, 3, device=DEV), 2), {}),
                 ((logits, scores.cpu(), 2), {}), ((logits.t().contiguous().t(), scores, 2), {}), ((logits, scores, 0), {}), ((logits, scores, 65), {}),
                 ((torch.zeros(33, 5, device=DEV), torch.zeros(1, 33, device=DEV), 2), {}), ((logits, scores, 2), dict(pad=50)), ((logits, scores, 2), dict(pad=-1)),
                 ((logits, scores, 2), dict(done=torch.zeros(2, 3, device=DEV))), ((logits, scores, 2), dict(done=torch.zeros(3, 2, dtype=torch.bool, device=DEV)))):
        with pytest.raises(ValueError):
            ops.beam_select(*a, **k)
    empty = ops.beam_select(logits[:0], scores[:0], 4)
    assert [tuple(x.shape) for x in empty] == [(0, 4)] * 3
    state, e = torch.zeros(2, 8, 5, device=DEV), err_word()
    for a in ((state[:, :, ::2], ints(range(6)), ints([[0] * 3] * 2)), (state, ints(range(5)), ints([[0] * 3] * 2)), (state, ints(range(6)).long(), ints([[0] * 3] * 2)),
              (state, ints(range(6)), ints([0] * 6)), (state, ints(range(6)), ints([[0] * 3] * 2).long()), (state.to(torch.int8), ints(range(6)), ints([[0] * 3] * 2)),
              (state, ints(range(33)), ints([[0] * 33])), (state.view(-1), ints(range(6)), ints([[0] * 3] * 2))):
        with pytest.raises(ValueError):
            ops.reorder_states(*a, e)
    pool, table, z, p = torch.zeros(2, 6, 1, 4, 8, device=DEV), ints([[x] for x in range(6)]), ints([0, 0]), ints([[0] * 3] * 2)
    for a in ((pool[..., :4], None, table, z, z, p), (pool, pool[:, :3], table, z, z, p), (pool, None, table[:5], z, z, p), (pool, None, table, z[:1], z, p),
              (pool, None, table, z, z.long(), p), (pool, None, table.view(-1), z, z, p), (pool[0, 0], None, table, z, z, p), (pool.to(torch.int8), None, table, z, z, p)):
        with pytest.raises(ValueError):
            ops.reorder_pages(*a, e)
    ops.reorder_states(state[:, :0], ints([]), ints(np.zeros((0, 3))), e)
    assert e.item() == 0
