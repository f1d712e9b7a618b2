"""Beam search through the engine against a search over the plain 64-bit model: scores of every place, sums of log probabilities of what
comes back, ends of sequence, prompts in portions, several prompts at once, windows (Padadra), and what it refuses."""
import dataclasses
import importlib
import re

import pytest
import torch

import plain_lfm2 as plain
from test_cli_gpu import run_tool
from tiny_configs import CONFIGS, make_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    d = tmp_path_factory.mktemp("models")
    return {name: make_model(d, name, "float32") for name in CONFIGS}


def log_probs(cfg, w, tokens):
    return torch.log_softmax(plain.forward(cfg, w, tokens).double(), -1)


def plain_search(cfg, w, prompt, K, steps, eos):
    """[(score, tokens, done)] of the K beams after `steps` tokens."""
    found = [(0.0, [], False)]
    for _ in range(steps):
        if all(d for _, _, d in found):
            break
        nxt = []
        for s, toks, d in found:
            if d:
                nxt.append((s, toks, True))
                continue
            lp = log_probs(cfg, w, prompt + toks)[-1]
            top = lp.topk(min(K, lp.numel()))
            nxt += [(s + float(v), toks + [int(t)], int(t) == eos) for v, t in zip(top.values, top.indices)]
        found = sorted(nxt, key=lambda f: -f[0])[:K]
    return found


def check(cfg, w, prompt, got, K, steps, eos, penalty=1.0):
    want = plain_search(cfg, w, prompt, K, steps, eos)
    assert len(got) == len(want)
    # 32-bit logits are off by 4e-6 of their size at most (tests/tolerances.py), a sum of log probabilities by twice that a token
    tol = 2 * 4e-6 * (1 + float(plain.forward(cfg, w, prompt).abs().max())) * steps + 1e-5
    assert sorted((b.score for b in got), reverse=True) == pytest.approx([s for s, _, _ in want], abs=tol)
    for b in got:
        lp = log_probs(cfg, w, prompt + b.tokens)
        assert b.score == pytest.approx(sum(float(lp[len(prompt) - 1 + i, t]) for i, t in enumerate(b.tokens)), abs=tol)
        assert b.finished == (eos is not None and b.tokens[-1] == eos) and (eos is None or eos not in b.tokens[:-1])
        assert len(b.tokens) == steps or b.finished
    ranks = [b.score / len(b.tokens) ** penalty for b in got]
    assert ranks == sorted(ranks, reverse=True) and len({tuple(b.tokens) for b in got}) == len(got)


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("graphs", [True, False])
def test_against_the_plain_model(folders, name, graphs):
    from cellm_b200 import Engine
    cfg, w = plain.load_folder(folders[name])
    eng = Engine(folders[name], dtype="float32", tokens_per_block=4, total_blocks=200, max_num_seqs=12, prefill_chunk=5, use_cuda_graphs=graphs, capture_after=1)
    prompts = [[5, 17, 3, 99, 250, 41, 8, 77, 60, 12, 1], [9]]
    out = eng.beam_search(prompts, beams=4, max_new_tokens=6, stop_eos=False)
    for p, got in zip(prompts, out):
        check(cfg, w, p, got, 4, 6, None)
    assert eng.stats()["free_pages"] == eng.stats()["total_pages"] and eng.stats()["free_slots"] == 12
    one = eng.beam_search(prompts[:1], beams=1, max_new_tokens=4, stop_eos=False)[0]
    check(cfg, w, prompts[0], one, 1, 4, None)


def test_a_beam_that_ends_stands(folders):
    """The end-of-sequence token is taken from what a search without one chose, so that beams end under way."""
    from cellm_b200 import Engine
    name = list(CONFIGS)[0]
    cfg, w = plain.load_folder(folders[name])
    eng = Engine(folders[name], dtype="float32", tokens_per_block=8, total_blocks=100, max_num_seqs=4)
    prompt = [7, 8, 200, 31]
    free = eng.beam_search([prompt], beams=4, max_new_tokens=5, stop_eos=False)[0]
    for eos in {free[0].tokens[1], free[1].tokens[2], free[0].tokens[0]}:
        eng.plan = dataclasses.replace(eng.plan, eos_token_id=eos)
        got = eng.beam_search([prompt], beams=4, max_new_tokens=5, length_penalty=0.6)[0]
        check(cfg, w, prompt, got, 4, 5, eos, 0.6)
        assert any(b.finished for b in got)


def test_fewer_tokens_than_beams(tmp_path):
    """A vocabulary of five tokens and eight beams: the first step finds five continuations, and beams that had none follow later."""
    from cellm_b200 import Engine
    name = list(CONFIGS)[0]
    folder = make_model(tmp_path, name, "float32", overrides={"vocab_size": 5, "eos_token_id": 4})
    cfg, w = plain.load_folder(folder)
    eng = Engine(folder, dtype="float32", tokens_per_block=4, total_blocks=100, max_num_seqs=8)
    prompt = [1, 0, 3, 2, 2, 1, 0]
    check(cfg, w, prompt, eng.beam_search([prompt], beams=8, max_new_tokens=5, stop_eos=False)[0], 8, 5, None)
    assert len(eng.beam_search([prompt], beams=8, max_new_tokens=1, stop_eos=False)[0]) == 5


def test_the_engine_serves_on_after_a_search(folders):
    from cellm_b200 import Engine, SamplingParams
    name = list(CONFIGS)[1]
    eng = Engine(folders[name], dtype="float32", tokens_per_block=8, total_blocks=100, max_num_seqs=8)
    prompts = [[3, 4, 5, 6], [100, 2, 7]]
    before = eng.generate(prompts, SamplingParams.greedy(8, stop_eos=False))
    found = eng.beam_search(prompts, beams=3, max_new_tokens=8, stop_eos=False)
    assert eng.generate(prompts, SamplingParams.greedy(8, stop_eos=False)) == before
    assert [b.tokens for b in eng.beam_search(prompts, beams=3, max_new_tokens=8, stop_eos=False)[0]] == [b.tokens for b in found[0]]


def test_windows_give_back_the_same_pages_of_all_beams(tmp_path):
    """A model with a windowed attention beside recurrent states: a pool that holds the beams only because pages in front of the window
    come back, with the same beams as a large pool gives, in either way of cutting the prompt."""
    from cellm_b200 import Engine, write_random_model
    from cellm_b200.config.presets import PADADRA_SHAPES
    import copy
    shape = copy.deepcopy(PADADRA_SHAPES["700m"][0])
    shape.update(vocab=400, width=64, layers=shape["layers"][1:4])
    for layer in shape["layers"]:
        m = layer["mixer"]
        if layer["type"] == "parallel":
            m["left"].update(heads=4, kv_heads=2, dim=16, vdim=16, mask={"size": 10}, rot={"base": 10000.0, "dims": 16})
            m["right"].update(heads=2, dim=16, vdim=16)
        else:
            m.update(heads=4, kv_heads=2, dim=16, vdim=16, decay_rank=8, gate_rank=8)
        layer["mlp"] = {"kind": "dense", "ff": 96}
    shape["embedding"]["bigram"].update(buckets=101)
    folder = write_random_model(str(tmp_path / "m"), shape, 3, "float32")
    prompt = [(7 * i) % 400 for i in range(61)]
    wide = Engine(folder, dtype="float32", tokens_per_block=4, total_blocks=400, max_num_seqs=4)
    want = wide.beam_search([prompt], beams=4, max_new_tokens=12, stop_eos=False)[0]
    tight = Engine(folder, dtype="float32", tokens_per_block=4, total_blocks=30, max_num_seqs=4, prefill_chunk=6)
    got = tight.beam_search([prompt], beams=4, max_new_tokens=12, stop_eos=False)[0]
    assert [b.score for b in got] == pytest.approx([b.score for b in want], abs=2e-3)
    assert tight.stats()["free_pages"] == tight.stats()["total_pages"]


@pytest.mark.parametrize("config", ["a", "b", "c", "d"])
@pytest.mark.parametrize("design", ["vezalorn", "tufadra", "padadra", "bozovik", "tikizen", "gonozen"])
def test_beams_of_every_design(tmp_path, design, config):
    """Caches of every kind in the order of the beams: what a search says of its beams is what one run over prompt and beam says. Either
    run is off by some 1e-5 of the logits' size (32 bits), a token's log probability by twice that: far below 2e-3 over nine tokens;
    a state or a row of another beam's moves a score by hundredths at least."""
    from cellm_b200 import Engine
    from cellm_b200.engine.step import StepEntry
    made = importlib.import_module(f"test_{design}_gpu")
    folder = made.write_model(tmp_path / "m", made.CONFIGS[config], 31)
    eng = Engine(folder, dtype="float32", tokens_per_block=8, total_blocks=160, max_num_seqs=10, prefill_chunk=16)
    V = eng.plan.vocab_size
    prompts = [[(11 * i + 5) % V for i in range(45)], [7 % V, 3 % V]]
    out = eng.beam_search(prompts, beams=5, max_new_tokens=9, stop_eos=False)
    assert eng.stats()["free_pages"] == eng.stats()["total_pages"]
    for prompt, found in zip(prompts, out):
        assert len(found) == 5 and len({tuple(b.tokens) for b in found}) == 5
        for n, b in enumerate(found):
            eng.cache.add(10 ** 6 + n)
            whole = prompt + b.tokens[:-1]
            lp = torch.log_softmax(eng.runner.run([StepEntry(10 ** 6 + n, whole, list(range(len(prompt) - 1, len(whole))))]).double(), -1)
            eng.cache.release(10 ** 6 + n)
            assert b.score == pytest.approx(float(lp[range(9), b.tokens].sum()), abs=2e-3)


@pytest.mark.parametrize("name", list(CONFIGS))
def test_finished_beams_need_no_pages(folders, name):
    """A pool that holds what the beams that go on read, and no more: the others' caches are given back. The same beams as a large pool
    gives."""
    from cellm_b200 import Engine
    cfg, w = plain.load_folder(folders[name])
    prompt, K, steps, ps = [7, 8, 200, 31, 90], 4, 24, 2
    make = lambda pages, eos: Engine(folders[name], dtype="float32", tokens_per_block=ps, total_blocks=pages, max_num_seqs=K)
    wide = make(400, None)
    free = wide.beam_search([prompt], beams=K, max_new_tokens=steps, stop_eos=False)[0]
    tried = 0
    for eos in dict.fromkeys(t for b in free for t in b.tokens[1:6]):
        wide.plan = dataclasses.replace(wide.plan, eos_token_id=eos)
        want = wide.beam_search([prompt], beams=K, max_new_tokens=steps)[0]
        # the beams that go on after each token, by a plain search
        need, found = 0, [(0.0, [], False)]
        for at in range(steps):
            nxt = []
            for s, toks, d in found:
                if d:
                    nxt.append((s, toks, True))
                    continue
                lp = log_probs(cfg, w, prompt + toks)[-1]
                top = lp.topk(K)
                nxt += [(s + float(v), toks + [int(t)], int(t) == eos) for v, t in zip(top.values, top.indices)]
            found = sorted(nxt, key=lambda f: -f[0])[:K]
            live = sum(not d for _, _, d in found)
            if not live:
                break
            if at + 1 < steps:
                need = max(need, live * (-(-(len(prompt) + at + 1) // ps)))
        need = max(need, -(-len(prompt) // ps))
        if need >= K * (-(-(len(prompt) + steps - 1) // ps)) - 2:
            continue
        tried += 1
        tight = make(need, eos)
        tight.plan = dataclasses.replace(tight.plan, eos_token_id=eos)
        got = tight.beam_search([prompt], beams=K, max_new_tokens=steps)[0]
        assert [b.tokens for b in got] == [b.tokens for b in want]
        check(cfg, w, prompt, got, K, steps, eos)
        assert tight.stats()["free_pages"] == tight.stats()["total_pages"] and tight.stats()["free_slots"] == K
    assert tried


@pytest.mark.parametrize("design", ["vezalorn", "tufadra", "padadra", "bozovik", "tikizen", "gonozen"])
def test_beams_that_end_in_every_design(tmp_path, design):
    """Caches of every kind given back by beams that end, beside another prompt's beams; scores as in the test above."""
    from cellm_b200 import Engine
    from cellm_b200.engine.step import StepEntry
    made = importlib.import_module(f"test_{design}_gpu")
    folder = made.write_model(tmp_path / "m", made.CONFIGS["a"], 31)
    eng = Engine(folder, dtype="float32", tokens_per_block=8, total_blocks=160, max_num_seqs=10, prefill_chunk=16)
    V = eng.plan.vocab_size
    prompts = [[(11 * i + 5) % V for i in range(45)], [7 % V, 3 % V]]
    free = eng.beam_search(prompts, beams=5, max_new_tokens=9, stop_eos=False)
    ended = 0
    for eos in dict.fromkeys(t for found in free for b in found for t in b.tokens[:4]):
        eng.plan = dataclasses.replace(eng.plan, eos_token_id=eos)
        out = eng.beam_search(prompts, beams=5, max_new_tokens=9)
        assert eng.stats()["free_pages"] == eng.stats()["total_pages"] and eng.stats()["free_slots"] == 10
        for prompt, found in zip(prompts, out):
            assert len(found) == 5 and len({tuple(b.tokens) for b in found}) == 5
            ended += sum(b.finished for b in found)
            for n, b in enumerate(found):
                assert b.finished == (b.tokens[-1] == eos) and eos not in b.tokens[:-1] and (b.finished or len(b.tokens) == 9)
                eng.cache.add(10 ** 6 + n)
                whole = prompt + b.tokens[:-1]
                lp = torch.log_softmax(eng.runner.run([StepEntry(10 ** 6 + n, whole, list(range(len(prompt) - 1, len(whole))))]).double(), -1)
                eng.cache.release(10 ** 6 + n)
                assert b.score == pytest.approx(float(lp[range(len(b.tokens)), b.tokens].sum()), abs=2e-3)
    assert ended


def test_refusals(folders):
    from cellm_b200 import Engine, SamplingParams
    from cellm_b200.cache.manager import OutOfPages
    name = list(CONFIGS)[0]
    eng = Engine(folders[name], dtype="float32", tokens_per_block=8, total_blocks=12, max_num_seqs=4)
    for bad in (dict(prompts=[[1]], beams=0), dict(prompts=[[1]], beams=33), dict(prompts=[[]]), dict(prompts=[[1, 10 ** 6]]), dict(prompts=[[1]], max_new_tokens=0),
                dict(prompts=[[1], [2]], beams=3), dict(prompts=[[1] * 250], max_new_tokens=10)):
        with pytest.raises(ValueError):
            eng.beam_search(**bad)
    assert eng.beam_search([]) == []
    with pytest.raises(OutOfPages):
        eng.beam_search([[1] * 40], beams=4, max_new_tokens=4)
    assert eng.stats()["free_pages"] == eng.stats()["total_pages"] and eng.stats()["free_slots"] == 4
    eng.add_request([1, 2], SamplingParams.greedy(2))
    with pytest.raises(RuntimeError):
        eng.beam_search([[1]])


def test_infer_prints_its_beams(folders):
    name = list(CONFIGS)[0]
    cfg, w = plain.load_folder(folders[name])
    out = run_tool("infer", "--model", folders[name], "--tokens", "5,17,3", "--gen", 4, "--beams", 3, "--dtype", "float32", "--stop-eos", "false")
    beams = [(float(s), [int(t) for t in ts.split(",")]) for s, ts in re.findall(r"^beam (-[\d.]+): ([\d,]+)$", out, re.M)]
    want = plain_search(cfg, w, [5, 17, 3], 3, 4, None)
    assert [s for s, _ in beams] == pytest.approx([s for s, _, _ in want], abs=1e-3) and all(len(t) == 4 for _, t in beams)
