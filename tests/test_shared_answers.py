"""Many answers to one prompt, as the operators for it are used together: the prompt runs once, its full pages are held by every answer
(CacheManager.fork), single-token steps read the shared keys once (shared_prefix_attention), and every answer's next token is chosen on
the device under rules of its own (sample with LogitRules, over the recorded texts).  Against the plain implementation, answer by answer.
"""
import functools
import random

import pytest
import torch

import plain_llama
from test_engine_rules import RulesBackend, under_rules
from test_engine import prompts_for
from torch_backend import TorchBackend, ref_perturbed

from mini_inference_engine_amd import SamplingParams
from mini_inference_engine_amd.cache import CacheAccountingError, CacheManager, GroupSpec
from mini_inference_engine_amd.engine.batch import KeptPlan, StepRow
from mini_inference_engine_amd.engine.runner import ModelRunner
from mini_inference_engine_amd.sampling import RuleInputs


# ---- pages that several requests hold

def test_a_forked_request_holds_the_full_pages():
    m = CacheManager(16, [GroupSpec(None, 20), GroupSpec(None, 20)], 6)
    a = m.open("a")
    assert m.reserve(a, 0, 50)
    b, c = m.fork(a, "b", 50), m.fork(a, "c", 15)
    assert b.tables == [t[:3] for t in a.tables] and c.tables == [[], []]
    m.check()
    assert m.num_free(0) == 19 - 4
    assert m.reserve(b, 48, 20) and m.num_free(0) == 19 - 6 and b.tables[0][3] not in a.tables[0]
    m.check()
    freed = []
    m.on_release = lambda g, pages: freed.extend((g, p) for p in pages)
    shared, own = list(a.tables[0][:3]), a.tables[0][3]
    m.close(a)
    assert [p for g, p in freed if g == 0] == [own]        # what b holds is not free
    m.check()
    d = m.fork(b, "d", 32)
    m.close(b)
    m.check()
    assert m.num_free(0) == 19 - 2 and d.tables[0] == shared[:2]
    m.close(c)
    m.close(d)
    m.check()
    assert m.num_free(0) == m.num_free(1) == 19


def test_what_cannot_be_forked():
    m = CacheManager(16, [GroupSpec(None, 20)], 4)
    a = m.open("a")
    m.reserve(a, 0, 20)
    for tokens in (48, -1):
        with pytest.raises(CacheAccountingError):
            m.fork(a, "b", tokens)
    with pytest.raises(CacheAccountingError):
        m.fork(a, "a", 16)
    m.check()
    assert "b" not in m.live
    m.close(a)
    with pytest.raises(CacheAccountingError):
        m.fork(a, "b", 16)
    windowed = CacheManager(16, [GroupSpec(None, 20), GroupSpec(32, 20)], 4)
    w = windowed.open("w")
    windowed.reserve(w, 0, 20)
    with pytest.raises(CacheAccountingError, match="windows"):
        windowed.fork(w, "x", 16)
    m.on_open = lambda slot: None
    a = m.open("a")
    m.reserve(a, 0, 20)
    with pytest.raises(CacheAccountingError, match="state"):
        m.fork(a, "b", 16)
    pool = m.pools[0]
    with pytest.raises(CacheAccountingError):
        pool.share([pool.free[0]])
    with pytest.raises(CacheAccountingError):
        pool.share([0])


@pytest.mark.parametrize("seed", range(6))
def test_no_page_lost_under_random_forks(seed):
    g = random.Random(seed)
    m = CacheManager(16, [GroupSpec(None, 40)], 12)
    live, n = {}, 0
    for _ in range(400):
        if live and g.random() < 0.35:
            name = g.choice(sorted(live))
            m.close(live.pop(name)[0])
        elif live and m.can_open() and g.random() < 0.5:
            rc, tokens = live[g.choice(sorted(live))]
            share = g.randint(0, tokens)
            n += 1
            live[n] = [m.fork(rc, n, share), share // 16 * 16]
        elif m.can_open():
            n += 1
            live[n] = [m.open(n), 0]
        for name in live:
            more = g.randint(0, 30)
            if m.reserve(live[name][0], live[name][1], more):
                live[name][1] += more
        m.check()
    for rc, _ in live.values():
        m.close(rc)
    m.check()
    assert m.num_free(0) == 39


# ---- the whole way

class SharedBackend(RulesBackend):
    """The kernel references, the shared keys read once only in name."""

    def plan_shared_prefix(self, groups, contexts, num_q_heads, num_kv_heads, head_dim, share=None):
        self._count("plan")
        return list(groups), list(contexts)

    def shared_prefix_attention(self, qkv, num_q_heads, num_kv_heads, head_dim, k_cache, v_cache, group, step, scale, plan, sink=None):
        self._count("shared")
        return self.paged_attention(qkv, num_q_heads, num_kv_heads, head_dim, k_cache, v_cache, group, step, scale, None, sink=sink)


ANSWERS = [SamplingParams(temperature=0.8, seed=1), SamplingParams(temperature=0.8, seed=2, repetition_penalty=1.5), SamplingParams(frequency_penalty=0.8),
           SamplingParams(temperature=1.2, seed=4, presence_penalty=0.6, logit_bias={3: 2.0}), SamplingParams(repetition_penalty=1.3)]


class Answer:
    """What the rules of a step look at (an engine's Sequence has the same)."""

    def __init__(self, i, cache, prompt, params):
        self.seq_id, self.cache, self.params, self.prompt_len, self.tokens = i, cache, params, len(prompt), list(prompt)

    output_ids = property(lambda self: self.tokens[self.prompt_len:])
    num_output_tokens = property(lambda self: len(self.tokens) - self.prompt_len)


def answers_to(m, device, dtype, slack, weights, prompt_tokens, steps=10, alone=2, graphs=False, share=None):
    """``alone``: of the answers, as many have another prompt, nothing shared.  ``share``: what the plans are asked for."""
    kw = dict(dtype=dtype, device=device, page_size=16, num_pages=60, max_step_tokens=256, max_rows=8)
    if device == "cpu":
        runner = ModelRunner(m["config"], backend=SharedBackend(torch.float32), weights=m["weights"], **kw)
    else:
        runner = ModelRunner(m["folder_f32"] if dtype == "float32" else m["folder_bf16"], **kw)
    if share is not None:
        runner.ops.plan_shared_prefix = functools.partial(runner.ops.plan_shared_prefix, share=share)
    if graphs:
        runner.capture_decode_graphs((1, 2, 4, 8), sample=True)
    history = runner.keep_token_history()
    prompt, other = prompts_for(m, [prompt_tokens, 19], seed=8)

    def run_prompt(name, ids):
        rc = runner.cache.open(name)
        assert runner.cache.reserve(rc, 0, len(ids))
        runner.forward_step([StepRow(rc, ids, 0)])
        return rc

    first = run_prompt("prompt", prompt[:-1])
    answers = []
    for i, params in enumerate(ANSWERS):
        if i < len(ANSWERS) - alone:
            rc = runner.fork(first, i, len(prompt) - 1)
            done = len(rc.tables[0]) * 16
            assert runner.cache.reserve(rc, done, len(prompt) + steps - done)
            if done < len(prompt) - 1:
                runner.forward_step([StepRow(rc, prompt[done:-1], done)])
            answers.append(Answer(i, rc, prompt, params))
        else:
            rc = run_prompt(i, other[:-1])
            assert runner.cache.reserve(rc, len(other) - 1, steps + 1)
            answers.append(Answer(i, rc, other, params))
    shared = (len(prompt) - 1) // 16 * 16
    runs = [(len(ANSWERS) - alone, shared)] + [(1, 0)] * alone
    runner.cache.check()
    inputs = RuleInputs(device, runner.vocab_size)
    for step in range(steps):
        rows = [StepRow(a.cache, [a.tokens[-1]], len(a.tokens) - 1, [0]) for a in answers]
        sampling = ([a.params.temperature for a in answers], [a.params.seed or 0 for a in answers], [a.num_output_tokens for a in answers])
        rules = inputs.make(answers, [len(a.tokens) for a in answers], history)
        logits = runner.forward_step(rows, sampling=sampling, rules=rules, shared_prefix=runs)
        assert runner.last_step_captured == (graphs and step > 0)
        chosen = runner.chosen_tokens[:len(answers)].tolist()
        if step == 0:                # the same step without sharing (its keys and values are written over with the same ones)
            again = runner.forward_step(rows, sampling=sampling, rules=rules)
            assert runner.last_step_captured == graphs
            assert float((logits - again).abs().max()) <= 2 * slack * float(again.abs().max())
        for a, tok, z in zip(answers, chosen, logits):
            want = plain_llama.forward(m["cfg"], m[weights], a.tokens)[-1]
            big = float(want.abs().max())
            assert float((z.cpu().double() - want.double()).abs().max()) <= slack * big
            score = ref_perturbed(under_rules(want, a.params, a.tokens[:a.prompt_len], a.output_ids, ()), a.params.temperature, a.params.seed or 0, step)
            stretch = max(a.params.repetition_penalty, 1.0) / (a.params.temperature or 1.0)
            assert float(score.max() - score[tok]) <= 2 * slack * big * stretch
            a.tokens.append(tok)
    assert len({tuple(a.output_ids) for a in answers}) == len(answers)        # the rules and seeds told them apart
    for a in answers:
        runner.cache.close(a.cache)
    runner.cache.close(first)
    runner.cache.check()
    return runner


@pytest.mark.parametrize("model", ["A", "B"])
@pytest.mark.parametrize("prompt_tokens", [49, 70, 12])
def test_answers_host(tiny_models, model, prompt_tokens):
    runner = answers_to(tiny_models[model], "cpu", "float32", 1e-5, "weights", prompt_tokens)
    assert runner.ops.calls["shared"] > 0 and runner.ops.calls["plan"] == 1       # one plan for all layers of ten steps


def test_a_plan_is_kept_as_long_as_it_fits(tiny_models, monkeypatch):
    m = tiny_models["A"]
    monkeypatch.setattr(KeptPlan, "AHEAD", 16)
    runner = ModelRunner(m["config"], backend=SharedBackend(torch.float32), weights=m["weights"], dtype="float32", device="cpu", num_pages=60,
                         page_size=16, max_step_tokens=256, max_rows=4)
    a, b, c = (runner.cache.open(x) for x in "abc")
    prompt = prompts_for(m, [40])[0]
    for rc in (a, c):
        assert runner.cache.reserve(rc, 0, runner.max_model_len)
        runner.forward_step([StepRow(rc, prompt, 0)])
    runner.cache.close(b)
    b = runner.cache.fork(a, "d", 40)
    assert runner.cache.reserve(b, 32, 100)
    runner.forward_step([StepRow(b, prompt[32:], 32)])

    def plans(starts, runs, first=a):
        before = runner.ops.calls.get("plan", 0)
        rows = [StepRow(rc, [1], s, [0]) for rc, s in zip((first, b, c), starts)]
        logits = runner.forward_step(rows, shared_prefix=runs)
        assert torch.allclose(logits, runner.forward_step(rows), atol=1e-5 * float(logits.abs().max()))
        return runner.ops.calls.get("plan", 0) - before

    runs, last = [(2, 32), (1, 0)], runner.max_model_len - 1
    assert plans((40, 40, 40), runs) == 1
    assert plans((41, 41, 41), tuple(runs)) == 0 and plans((56, 41, 56), runs) == 0
    assert plans((57, 41, 40), runs) == 1                       # a row beyond what was planned
    assert plans((57, 41, 40), [(2, 16), (1, 0)]) == 1          # other runs
    assert plans((57, 41, 40), runs) == 1
    assert plans((40, 40, 40), runs) == 1                       # a row far short of what was planned
    assert plans((40, 40), [(2, 32)]) == 1
    assert plans((last, 100, last), runs) == 1                  # planned no further than the block tables go


def test_refused_shared_steps(tiny_models):
    m = tiny_models["A"]
    runner = ModelRunner(m["config"], backend=SharedBackend(torch.float32), weights=m["weights"], dtype="float32", device="cpu", num_pages=40,
                         max_step_tokens=64, max_rows=4)
    prompt = prompts_for(m, [40])[0]
    a = runner.cache.open("a")
    runner.cache.reserve(a, 0, 60)
    runner.forward_step([StepRow(a, prompt, 0)])
    b = runner.cache.fork(a, "b", 40)
    runner.cache.reserve(b, 32, 30)
    runner.forward_step([StepRow(b, prompt[32:], 32)])
    rows = [StepRow(a, [1], 40, [0]), StepRow(b, [1], 40, [0])]
    runner.forward_step(rows, shared_prefix=[(2, 32)])
    for bad in ([(2, 48)], [(2, 40)], [(1, 32)], [(3, 0)], [(2, -16)], [(0, 0), (2, 32)]):
        with pytest.raises(ValueError):
            runner.forward_step(rows, shared_prefix=bad)
    other = runner.cache.open("c")
    runner.cache.reserve(other, 0, 60)
    with pytest.raises(ValueError, match="same pages"):
        runner.forward_step([rows[0], StepRow(other, [1], 40, [0])], shared_prefix=[(2, 32)])
    with pytest.raises(ValueError, match="single tokens"):
        runner.forward_step([rows[0], StepRow(b, [1, 2], 40, [0])], shared_prefix=[(2, 32)])


@pytest.mark.gpu
@pytest.mark.parametrize("graphs, share", [(False, None), (True, True), (False, True)])
@pytest.mark.parametrize("model", ["A", "B", "C"])
@pytest.mark.parametrize("dtype, slack, weights", [("float32", 1e-5, "weights"), ("bfloat16", 2e-2, "weights_bf16")])
def test_answers_gpu(tiny_models, model, dtype, slack, weights, graphs, share):
    answers_to(tiny_models[model], "cuda", dtype, slack, weights, 70, graphs=graphs, share=share)


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["A", "B", "C"])
@pytest.mark.parametrize("dtype, slack, weights", [("float32", 1e-5, "weights"), ("bfloat16", 2e-2, "weights_bf16")])
def test_captured_steps_of_shared_first_parts(tiny_models, monkeypatch, model, dtype, slack, weights):
    """Steps replayed under kept plans are what they are kernel by kernel, over new plans, other rows, rows without wishes and back."""
    m = tiny_models[model]
    monkeypatch.setattr(KeptPlan, "AHEAD", 5)
    runner = ModelRunner(m["folder_f32"] if dtype == "float32" else m["folder_bf16"], dtype=dtype, num_pages=60, page_size=16, max_step_tokens=256,
                         max_rows=8)
    runner.capture_decode_graphs((2, 8), sample=True)
    runner.ops.plan_shared_prefix = functools.partial(runner.ops.plan_shared_prefix, share=True)
    prompt = prompts_for(m, [49], seed=3)[0]
    first = runner.cache.open("p")
    assert runner.cache.reserve(first, 0, 49)
    runner.forward_step([StepRow(first, prompt[:48], 0)])
    caches = [runner.fork(first, i, 48) for i in range(4)]
    for rc in caches:
        assert runner.cache.reserve(rc, 48, 40)

    def step(k, who, runs, want=None, sample=True):
        rows = [StepRow(caches[i], [7 + 3 * i + k], 48 + k, [] if want is not None and i not in want else [0]) for i in who]
        n = sum(len(r.want) for r in rows)
        sampling = ([0.7] * n, list(range(n)), [k] * n) if sample else None
        got = runner.forward_step(rows, sampling=sampling, shared_prefix=runs)
        captured, chosen = runner.last_step_captured, runner.chosen_tokens[:n].tolist()
        if got is not None:
            got = got.clone()
        graphs, runner.graphs = runner.graphs, None
        want_logits = runner.forward_step(rows, sampling=sampling, shared_prefix=runs)
        runner.graphs = graphs
        if got is None:
            assert want_logits is None
        else:
            # (the step kernel by kernel may split a matrix product otherwise than a captured one)
            assert got.shape == want_logits.shape and float((got - want_logits).abs().max()) <= slack * float(want_logits.abs().max())
            if sample and torch.equal(got, want_logits):
                assert chosen == runner.chosen_tokens[:n].tolist()
        return captured

    runs = [(3, 48), (1, 0)]
    assert [step(k, range(4), runs) for k in range(5)] == [False, True, True, True, True]
    graph = runner.shared_graph
    assert step(5, range(4), runs) and runner.shared_graph is graph
    assert not step(6, range(4), runs) and step(7, range(4), runs) and runner.shared_graph is not graph       # beyond what was planned
    assert not step(8, (0, 2), [(2, 48)]) and step(8, (0, 2), [(2, 48)])
    assert step(9, (0, 2), [(2, 48)], want=(2,), sample=False) and step(9, (0, 2), [(2, 48)], want=(), sample=False)
    assert not step(9, (0, 2), [(2, 48)], want=(2,))                   # choices for some rows only: kernel by kernel
    assert not step(10, range(4), runs) and step(11, range(4), tuple(runs))
    for rc in [first, *caches]:
        runner.cache.close(rc)
    runner.cache.check()
