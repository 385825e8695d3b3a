"""Texts that rules on logits look at, in every order in which they can come to be kept: a request forked from one that ran before the
texts were, forked before they were, forked past the runner; and pages with and without the text they hold.  On the CPU, on the kernel
references, against the plain implementation.
"""
import pytest
import torch

import plain_llama
from test_engine import prompts_for
from test_engine_rules import under_rules
from test_shared_answers import Answer, SharedBackend
from torch_backend import ref_perturbed

from mini_inference_engine_amd import SamplingParams
from mini_inference_engine_amd.engine.batch import StepRow
from mini_inference_engine_amd.engine.runner import ModelRunner
from mini_inference_engine_amd.sampling import RuleInputs

PENALTIES = SamplingParams(repetition_penalty=1.7, frequency_penalty=0.4, presence_penalty=0.3)


def runner_of(m, **kw):
    return ModelRunner(m["config"], backend=SharedBackend(torch.float32), weights=m["weights"], dtype="float32", device="cpu", num_pages=60,
                       page_size=16, max_step_tokens=256, max_rows=8, **kw)


def run_prompt(runner, name, ids):
    rc = runner.cache.open(name)
    assert runner.cache.reserve(rc, 0, len(ids) + 8)
    runner.forward_step([StepRow(rc, ids, 0)])
    return rc


def next_token(runner, answer, m):
    """The answer's next token under its rules, checked against the definition."""
    inputs = RuleInputs(runner.device, runner.vocab_size)
    done = answer.cache.recorded if runner.token_history is not None else None
    start = len(answer.tokens) - 1
    rules = inputs.make([answer], [len(answer.tokens)], runner.token_history)
    runner.forward_step([StepRow(answer.cache, [answer.tokens[-1]], start, [0])], sampling=([0.0], [0], [0]), rules=rules)
    tok = int(runner.chosen_tokens[0])
    want = plain_llama.forward(m["cfg"], m["weights"], answer.tokens)[-1]
    score = ref_perturbed(under_rules(want, answer.params, answer.tokens[:answer.prompt_len], answer.output_ids, ()), 0.0, 0, 0)
    assert float(score.max() - score[tok]) <= 1e-5 * float(want.abs().max()) * answer.params.repetition_penalty, (tok, int(score.argmax()), done)
    answer.tokens.append(tok)


def test_a_fork_of_a_request_that_ran_before_the_texts_were_kept(tiny_models):
    m = tiny_models["A"]
    runner = runner_of(m)
    prompt = prompts_for(m, [49], seed=3)[0]
    first = run_prompt(runner, "p", prompt[:-1])
    history = runner.keep_token_history()
    with pytest.raises(ValueError, match="text"):
        runner.fork(first, "a", 48)
    runner.cache.check()
    assert "a" not in runner.cache.live
    with pytest.raises(ValueError, match="text"):
        runner.fork(first, "a", 48, text=prompt[:47])
    a = runner.fork(first, "a", 48, text=prompt)
    assert history[a.state_slot, :48].tolist() == prompt[:48]
    assert runner.cache.reserve(a, 48, 8)
    answer = Answer(0, a, prompt, PENALTIES)
    for _ in range(4):
        next_token(runner, answer, m)
    # a fork of the fork has what that has
    b = runner.fork(a, "b", 50)
    assert history[b.state_slot, :48].tolist() == prompt[:48]
    # one that shares nothing needs no text
    c = runner.fork(first, "c", 15)
    assert c.tables == [[]]


def test_a_part_of_the_text_was_kept(tiny_models):
    """The prompt's first portion ran before the texts were kept: its second is there, but nothing from the beginning is."""
    m = tiny_models["A"]
    runner = runner_of(m)
    prompt = prompts_for(m, [60], seed=4)[0]
    first = runner.cache.open("p")
    assert runner.cache.reserve(first, 0, 60)
    runner.forward_step([StepRow(first, prompt[:20], 0)])
    runner.keep_token_history()
    runner.forward_step([StepRow(first, prompt[20:], 20)])
    with pytest.raises(ValueError, match="text"):
        runner.fork(first, "a", 48)
    runner.forward_step([StepRow(first, prompt[:20], 0)])          # run again from its beginning: kept as far as that goes
    assert runner.fork(first, "b", 16).recorded == 16
    with pytest.raises(ValueError, match="text"):
        runner.fork(first, "c", 32)


def test_a_fork_from_before_the_texts_were_kept(tiny_models):
    """Its first step comes later, its shared tokens' did not: penalties are refused, other rules are not."""
    m = tiny_models["A"]
    runner = runner_of(m)
    prompt = prompts_for(m, [49], seed=3)[0]
    first = run_prompt(runner, "p", prompt[:-1])
    early = runner.fork(first, "a", 48)
    assert runner.cache.reserve(early, 48, 8)
    history = runner.keep_token_history()
    inputs = RuleInputs(runner.device, runner.vocab_size)
    fresh = run_prompt(runner, "q", prompt[:-1])
    late = runner.fork(fresh, "b", 48)
    assert runner.cache.reserve(late, 48, 8)
    past = runner.cache.fork(fresh, "c", 48)                       # not by the runner: the pages without their text
    assert runner.cache.reserve(past, 48, 8)
    for bad in (early, past):
        answers = [Answer(0, late, prompt, PENALTIES), Answer(1, bad, prompt, PENALTIES)]
        rows = [StepRow(a.cache, prompt[-1:], 48, [0]) for a in answers]
        rules = inputs.make(answers, [49, 49], history)
        before = late.recorded, history.clone()
        with pytest.raises(ValueError, match="text"):
            runner.forward_step(rows, sampling=([0.0] * 2, [0] * 2, [0] * 2), rules=rules)
        assert late.recorded == before[0] and torch.equal(history, before[1])
        answers[1].params = SamplingParams(logit_bias={3: 100.0})
        rules = inputs.make(answers, [49, 49], history)
        runner.forward_step(rows, sampling=([0.0] * 2, [0] * 2, [0] * 2), rules=rules)
        assert int(runner.chosen_tokens[1]) == 3
    # a row without wishes has no rules: the second row of logits is the third row's
    rows = [StepRow(late, prompt[-1:], 48, [0]), StepRow(past, prompt[-1:], 48, []), StepRow(fresh, prompt[-1:], 48, [0])]
    answers = [Answer(0, late, prompt, PENALTIES), Answer(1, fresh, prompt, PENALTIES)]
    runner.forward_step(rows, sampling=([0.0] * 2, [0] * 2, [0] * 2), rules=inputs.make(answers, [49, 49], history))


def test_a_slot_that_was_another_requests(tiny_models):
    """What a request before left in the slot's row is not the text of the one that has it now."""
    m = tiny_models["A"]
    runner = runner_of(m, num_state_slots=3)
    runner.keep_token_history()
    prompt, other = prompts_for(m, [49, 60], seed=5)
    first = run_prompt(runner, "p", other)
    slot = first.state_slot
    runner.cache.close(first)
    second = run_prompt(runner, "q", prompt[:-1])
    again = runner.cache.open("r")
    assert slot in (second.state_slot, again.state_slot)
    runner.cache.close(again)
    a = runner.fork(second, "a", 48)
    assert runner.token_history[a.state_slot, :48].tolist() == prompt[:48]
    assert runner.cache.reserve(a, 48, 8)
    answer = Answer(0, a, prompt, PENALTIES)
    for _ in range(3):
        next_token(runner, answer, m)


@pytest.mark.gpu
def test_forks_with_their_text_gpu(tiny_models):
    m = tiny_models["A"]
    runner = ModelRunner(m["folder_f32"], dtype="float32", num_pages=60, page_size=16, max_step_tokens=256, max_rows=8)
    prompt = prompts_for(m, [49], seed=3)[0]
    first = run_prompt(runner, "p", prompt[:-1])
    history = runner.keep_token_history()
    with pytest.raises(ValueError, match="text"):
        runner.fork(first, "a", 48)
    a = runner.fork(first, "a", 48, text=prompt)
    b = runner.fork(a, "b", 48)
    for rc in (a, b):
        assert history[rc.state_slot, :48].tolist() == prompt[:48]
        assert runner.cache.reserve(rc, 48, 8)
        answer = Answer(0, rc, prompt, PENALTIES)
        for _ in range(3):
            next_token(runner, answer, m)
