"""Scored prompts and told log probabilities inside the engine, on the GPU: the operators of ``ops.token_logprobs`` and
``ops.head_logprobs`` as the step function, the engine and the command line use them."""
import math

import numpy as np
import pytest
import torch

import plain_qwen3 as P
from helpers import TINY, make_model_folder, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("score_models")
    return {n: make_model_folder(n, str(root)) for n in TINY}


def engine(folders, name, dtype="float32", **kw):
    import airun_b200
    o = dict(page_size=TINY[name]["page_size"], cache_tokens=768, max_batch_tokens=48, max_requests=4)
    return airun_b200.Engine.from_folder(folders[name], dtype=dtype, **{**o, **kw})


def from_logits(x, tokens):
    """Log probabilities, entropies and tokens in descending order of their logits, in 64 bits."""
    lp = torch.log_softmax(x.double(), dim=-1)
    t = torch.as_tensor(tokens)
    return lp.gather(1, t[:, None])[:, 0], -(lp.exp() * lp).sum(1), lp


# A logit of these models is off by about 2e-5 between two ways through the layers in float32 (sums of up to 512 products of size 1, 24 layers'
# roundings at most); a log probability by twice that, an entropy by 2 ln V times.  In bfloat16 both sides read the same hidden states, and
# sums of up to 256 products are off by 2^-23 * 16 steps of what they add up to (about 3).
TOL = 4e-5 * 2 * math.log(512)


@pytest.mark.parametrize("name", list(TINY))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scored_places_agree_with_their_logits(name, dtype, folders):
    """Portions, single tokens and requests that want nothing in one batch; both ways from the same cache."""
    from airun_b200 import StepEntry
    eng = engine(folders, name, dtype)
    V = eng.config.vocab_size
    toks = [random_tokens(n, V, 7 + n) for n in (21, 1, 9)]
    want = [(0, 3, 4, 20), (0,), ()]
    targets = [5, -1, V, 0, V - 1]
    for r in "abc":
        eng.manager.add_request(r)
    entries = [StepEntry(r, t, w) for r, t, w in zip("abc", toks, want)]
    logits = eng.runner.step(entries).float().cpu()
    for r in "abc":
        eng.manager.free_request(r)
        eng.manager.add_request(r)
    for top in (0, 3, 20):
        got = eng.runner.score(entries, targets, top)
        lp, H, all_lp = from_logits(logits, [t if 0 <= t < V else 0 for t in targets])
        assert got.logprob.shape == (5,) and got.logprob[[1, 2]].tolist() == [-math.inf] * 2
        keep = [0, 3, 4]
        assert float((got.logprob.cpu()[keep].double() - lp[keep]).abs().max()) < TOL
        assert float((got.entropy.cpu().double() - H).abs().max()) < TOL
        if top:
            ids = got.top_ids.cpu().long()
            assert ids.shape == (5, top)
            assert float((got.top_logprobs.cpu().double() - all_lp.gather(1, ids)).abs().max()) < TOL
            assert float((all_lp.topk(top, dim=1).values - all_lp.gather(1, ids)).abs().max()) < TOL      # the largest, but for near ties
            assert all(len(set(row)) == top for row in ids.tolist())
        for r in "abc":
            eng.manager.free_request(r)
            eng.manager.add_request(r)
    assert eng.runner.score([StepEntry("a", toks[0])], []) is None
    eng.runner.raise_on_device_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("design,shape", [("losalorn", "l1"), ("losalorn", "l2"), ("tagulix", "t1"), ("tagulix", "t4"), ("gamanex", "g1")])
def test_other_designs_are_scored(design, shape, dtype, tmp_path):
    """A capped head, a residual of several streams, a head of a model with its own norm: portions of two requests against the step's logits."""
    import importlib
    from airun_b200 import Engine, StepEntry
    t = importlib.import_module("test_" + design)
    make, page = t.SHAPES[shape][:2]
    cfg = make()
    more = {"rel_rows": t.SHAPES[shape][2]} if len(t.SHAPES[shape]) > 2 else {}
    folder = t.P.write_folder(str(tmp_path), cfg, t.P.random_weights(cfg, seed=5, **more))
    eng = Engine.from_folder(folder, dtype=dtype, page_size=page, cache_tokens=512, max_batch_tokens=128, max_requests=4, max_context=512)
    V = eng.config.vocab_size
    toks = [random_tokens(n, V, n) for n in (30, 13)]
    entries = [StepEntry(r, s, range(len(s))) for r, s in zip("ab", toks)]
    targets = [x for s in toks for x in s[1:] + s[:1]]

    def fresh():
        for r in "ab":
            if r in eng.manager.requests:
                eng.manager.free_request(r)
            eng.manager.add_request(r)

    fresh()
    lp, H, all_lp = from_logits(eng.runner.step(entries).float().cpu(), targets)
    fresh()
    got = eng.runner.score(entries, targets, 3)
    eng.runner.raise_on_device_error()
    assert float((got.logprob.cpu().double() - lp).abs().max()) < TOL and float((got.entropy.cpu().double() - H).abs().max()) < TOL
    assert float((got.top_logprobs.cpu().double() - all_lp.gather(1, got.top_ids.cpu().long())).abs().max()) < TOL


def test_score_refuses_what_step_refuses(folders):
    from airun_b200 import StepEntry
    from airun_b200.engine.step import StepError
    eng = engine(folders, "A")
    eng.manager.add_request("a")
    with pytest.raises(StepError, match="targets"):
        eng.runner.score([StepEntry("a", [1, 2], (0, 1))], [3])
    with pytest.raises(StepError, match="alternatives"):
        eng.runner.score([StepEntry("a", [1, 2], (0,))], [3], top=129)
    with pytest.raises(StepError, match="place"):
        eng.runner.score([StepEntry("a", [1, 2], (2,))], [3])
    assert eng.manager.get("a").num_tokens == 0


@pytest.mark.parametrize("name", list(TINY))
def test_scored_prompts_are_the_plain_implementations(name, folders):
    """Prompts longer than a step, of one token, and more of them than requests fit."""
    cfg, W = P.read_model_folder(folders[name])
    eng = engine(folders, name, max_batch_tokens=32, max_requests=3)
    longest = min(120, cfg["max_position_embeddings"] - 1)
    prompts = [random_tokens(n, cfg["vocab_size"], 30 + n) for n in (longest, 1, 33, 2, 17, 32)]
    got = eng.score(prompts, top=2)
    for p, s in zip(prompts, got):
        assert s.token_ids == p and s.logprobs[0] is None and s.entropies[0] is None and s.top[0] == []
        assert len(s.logprobs) == len(s.entropies) == len(s.top) == len(p)
        if len(p) > 1:
            lp, H, all_lp = from_logits(P.plain_forward(cfg, W, p, torch.float32)[:-1], p[1:])
            assert np.abs(np.array(s.logprobs[1:]) - lp.numpy()).max() < TOL
            assert np.abs(np.array(s.entropies[1:]) - H.numpy()).max() < TOL
            assert abs(s.total - float(lp.sum())) < TOL * len(p)
            for row, pairs in zip(all_lp, s.top[1:]):
                assert len(pairs) == 2 and all(abs(float(row[t]) - v) < TOL for t, v in pairs) and pairs[0][1] >= pairs[1][1]
                assert float(row.max()) - float(row[pairs[0][0]]) < TOL
    one = eng.score(prompts[2])
    assert one.top == [[]] * 33 and np.abs(np.array(one.logprobs[1:]) - np.array(got[2].logprobs[1:])).max() < TOL
    assert eng.manager.free_pages() == {g.gid: eng.manager.num_pages for g in eng.manager.paged} and not eng.manager.requests
    eng.manager.check_invariants()


def test_scoring_between_requests(folders):
    """A small pool, kept caches that have to go, and requests before and after."""
    import airun_b200
    eng = engine(folders, "B", page_size=8, num_pages=10, cache_tokens=None, max_context=72, prefix_cache=True, max_requests=2)
    V = eng.config.vocab_size
    prompts = [random_tokens(n, V, n) for n in (40, 41, 72)]
    before = eng.generate(prompts[0], airun_b200.SamplingParams.greedy(), max_new_tokens=8).token_ids
    scores = eng.score(prompts)
    alone = engine(folders, "B", page_size=8)
    for p, s in zip(prompts, scores):
        assert np.abs(np.array(s.logprobs[1:]) - np.array(alone.score(p).logprobs[1:])).max() < TOL
    assert eng.generate(prompts[0], airun_b200.SamplingParams.greedy(), max_new_tokens=8).token_ids == before
    with pytest.raises(ValueError, match="context"):
        eng.score(random_tokens(74, V, 1))
    with pytest.raises(ValueError, match="outside"):
        eng.score([1, V])
    with pytest.raises(ValueError, match="empty"):
        eng.score([[1, 2], []])
    with pytest.raises(ValueError, match="top"):
        eng.score([1, 2], top=129)
    assert eng.score([]) == []
    eng.add_request(prompts[0], airun_b200.SamplingParams.greedy(), max_new_tokens=2)
    with pytest.raises(RuntimeError, match="running or waiting"):
        eng.score(prompts[1])
    while eng.has_work():
        eng.run_step()
    eng.manager.check_invariants()


def settings():
    from airun_b200 import SamplingParams as S
    return [dict(S.greedy().__dict__, logprobs=0), dict(S.temperature_only(0.9, 4).__dict__, logprobs=3),       # the host draws from the whole row
            dict(S(seed=3).__dict__, logprobs=5),                                            # the usual chain: its candidates travel
            dict(S(seed=5, temperature=0.7, top_p=0.9, repeat_penalty=1.0).__dict__, logprobs=2), dict(S.greedy().__dict__),
            dict(S(seed=6, logit_bias=((3, 2.0),)).__dict__, logprobs=1),                    # the whole row travels
            dict(S(seed=7, top_k=1).__dict__, logprobs=200)]                                 # more than are told: the whole row


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("how", ["told", "distrusted"])
def test_told_log_probabilities_are_those_of_whole_rows(dtype, how, folders, monkeypatch):
    """The same tokens as with every row on the host, and log probabilities that differ by float32 roundings of two formulas only (values of size
    20 and their sums: a few units of 2^-20)."""
    from airun_b200 import SamplingParams
    params = settings()
    results = {}
    for mode in ("0", "1"):
        monkeypatch.setenv("AIRUN_NARROW_ROWS", mode)
        eng = engine(folders, "D", dtype, max_batch_tokens=64, max_requests=8)
        eng._distrust_candidates = how == "distrusted" and mode == "1"
        prompts = [random_tokens(5 + 7 * i, eng.config.vocab_size, 60 + i) for i in range(len(params))]
        results[mode] = eng.generate(prompts, [SamplingParams(**p) for p in params], max_new_tokens=10)
    for p, a, b in zip(params, results["0"], results["1"]):
        assert a.token_ids == b.token_ids
        if p["logprobs"] is None:
            assert a.logprobs is None and b.logprobs is None
            continue
        assert len(b.logprobs) == 10
        for x, y in zip(a.logprobs, b.logprobs):
            assert x.token == y.token and abs(x.logprob - y.logprob) < 1e-5
            assert [t for t, _ in x.top] == [t for t, _ in y.top] and len(y.top) == min(p["logprobs"], 512)
            assert all(abs(u - v) < 1e-5 for (_, u), (_, v) in zip(x.top, y.top))


def test_a_head_of_its_own_is_scored_from_its_logits(folders):
    """A part that only forms logits is scored too, by way of them."""
    from airun_b200 import StepEntry
    from airun_b200.parts.base import Head
    eng = engine(folders, "B", "bfloat16")
    toks = random_tokens(30, eng.config.vocab_size, 3)
    entry = [StepEntry("a", toks, range(30))]
    got = []
    for plain in (False, True):
        if plain:
            own = eng.model.head
            eng.model.head.score = lambda *a: Head.score(own, *a)
        eng.manager.add_request("a")
        got.append(eng.runner.score(entry, toks[1:] + [0], 4))
        eng.manager.free_request("a")
    a, b = got
    assert float((a.logprob - b.logprob).abs().max()) < TOL and float((a.entropy - b.entropy).abs().max()) < TOL
    assert float((a.top_logprobs - b.top_logprobs).abs().max()) < TOL


def test_a_drawn_token_has_the_value_of_its_entry_among_the_alternatives(folders):
    """A token that the host draws from its candidates, or the device picks, and that is among the alternatives too has one value, bit for bit; one that is not, and a
    draw without alternatives, the value that the same draw has where it is listed."""
    from airun_b200 import SamplingParams as S
    draws = [dict(S(seed=3).__dict__), dict(S(seed=5, temperature=0.7, top_p=0.9, repeat_penalty=1.0).__dict__), dict(S(seed=11, temperature=3.0, top_k=60).__dict__),
             dict(S.greedy().__dict__), dict(S(temperature=0.0, repeat_penalty=1.3).__dict__)]
    eng = engine(folders, "D", max_batch_tokens=64, max_requests=8)
    prompts = [random_tokens(5 + 7 * i, eng.config.vocab_size, 80 + i) for i in range(len(draws))]
    results = {}
    for told in (0, 1, 100):
        results[told] = eng.generate(prompts, [S(**dict(p, logprobs=told)) for p in draws], max_new_tokens=12)
    listed = 0
    for few, one, many in zip(results[0], results[1], results[100]):
        assert few.token_ids == one.token_ids == many.token_ids
        for a, b, c in zip(few.logprobs, one.logprobs, many.logprobs):
            assert a.top == [] and len(b.top) == 1 and len(c.top) == 100 and b.top[0] == c.top[0]
            assert a.logprob == b.logprob == c.logprob
            entry = dict(c.top).get(c.token)
            if entry is not None:
                listed += 1
                assert c.logprob == entry
    assert listed > 30


@pytest.mark.parametrize("batched", [[], ["--chunk", "20", "--batched"]])
def test_perplexity_shows_a_broken_model_and_refuses_ids_it_does_not_have(batched, folders, tmp_path, monkeypatch, capsys):
    """One logit that is not a number is a loss that is not one, and so is the mean; a last id behind the vocabulary ends the command."""
    import airun_b200
    from airun_b200.cli import main
    V = engine(folders, "B").config.vocab_size
    f = tmp_path / "ids.txt"
    f.write_text(" ".join(map(str, random_tokens(40, V, 8))))
    args = ["perplexity", folders["B"], "-f", str(f), "--dtype", "float32"] + batched
    assert main(args) == 0
    sound = capsys.readouterr().out
    assert "not finite" not in sound and "nan" not in sound
    load = airun_b200.Engine.from_folder

    def broken(*a, **k):
        eng = load(*a, **k)
        eng.model.head.weight = eng.model.head.weight.clone()
        eng.model.head.weight[7, 3] = math.nan
        return eng

    monkeypatch.setattr(airun_b200.Engine, "from_folder", broken)
    assert main(args + ["--worst", "1"]) == 0
    out = capsys.readouterr().out
    n = 18 if batched else 39
    assert "mean loss   nan" in out and f"the losses of {n} of the {n} tokens" in out
    monkeypatch.setattr(airun_b200.Engine, "from_folder", load)
    f.write_text(f.read_text() + f" {V}")
    with pytest.raises(SystemExit, match="outside"):
        main(["perplexity", folders["B"], "-f", str(f), "--dtype", "float32"])


def test_targets_far_outside_the_vocabulary_ask_for_none(folders):
    """Ids that 32 bits do not hold are ids outside the vocabulary like any other."""
    from airun_b200 import StepEntry
    eng = engine(folders, "A")
    V = eng.config.vocab_size
    eng.manager.add_request("a")
    got = eng.runner.score([StepEntry("a", [1, 2, 3, 4, 5, 6], range(6))], [2, 1 << 40, -1 << 40, V, (1 << 32) + 2, np.int64(3)])
    lp = got.logprob.tolist()
    assert lp[1:5] == [-math.inf] * 4 and math.isfinite(lp[0]) and math.isfinite(lp[5])
    eng.manager.free_request("a")
    eng.runner.raise_on_device_error()
