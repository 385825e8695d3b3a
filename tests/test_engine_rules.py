"""Requests with rules on their logits through the engine's entry point: penalties, biases and allowed tokens, against the plain
implementation of the model and of the rules.  Without a GPU the engine's host logic runs on the kernel references; with one, on the
HIP kernels.  A token is accepted if its score under the rules is within ``slack`` of the best one (as in test_engine.py).
"""
import math

import pytest
import torch

import plain_llama
from test_engine import prompts_for
from test_logit_rules import plain as plain_rules, recorded
from torch_backend import TorchBackend, ref_perturbed, ref_sample

from mini_inference_engine_amd import LLMEngine, SamplingParams
from mini_inference_engine_amd.config import EngineConfig
from mini_inference_engine_amd.sampling.rules import mask_words


class RulesBackend(TorchBackend):
    """The kernel references with the rules among them."""

    def record_tokens(self, history, step):
        self._count("record_tokens")
        history.copy_(recorded(history, step))

    def adjust_logits(self, logits, rules, out=None):
        y = plain_rules(logits, rules)[0].float()
        return y if out is None else out.copy_(y)

    def sample(self, logits, temperatures, seeds, counters, out=None, rules=None):
        if rules is None:
            return super().sample(logits, temperatures, seeds, counters, out=out)
        self._count("sample under rules")
        tokens = ref_sample(self.adjust_logits(logits, rules), temperatures, seeds, counters)
        return tokens if out is None else out.copy_(tokens)


def engine(m, device, dtype, **cfg):
    if device == "cpu":
        return LLMEngine(m["config"], EngineConfig(**cfg), dtype=dtype, verbose=False, device="cpu", backend=RulesBackend(torch.float32),
                         weights=m["weights"])
    return LLMEngine(m["folder_f32"] if dtype == "float32" else m["folder_bf16"], EngineConfig(**cfg), dtype=dtype, verbose=False)


def under_rules(z, sp, prompt, output, stop):
    """The definition, one token after another, in 64 bits."""
    z = z.double().clone()
    for t in set(prompt) | set(output):
        z[t] = z[t] / sp.repetition_penalty if z[t] > 0 else z[t] * sp.repetition_penalty
    for t in set(output):
        z[t] -= sp.frequency_penalty * output.count(t) + sp.presence_penalty
    for t, b in (sp.logit_bias or {}).items():
        z[t] += b
    allowed = sp.allowed_tokens(list(output)) if sp.allowed_tokens else None
    if allowed is not None:
        allowed = list(allowed) or sorted(stop)
        hidden = torch.ones(z.shape[0], dtype=torch.bool)
        hidden[allowed] = False
        z[hidden] = -math.inf
    return z


def check(m, eng, prompts, outs, params, slack_rel, weights="weights"):
    for prompt, out, sp in zip(prompts, outs, params):
        done = []
        for i, tok in enumerate(out.output_ids):
            logits = plain_llama.forward(m["cfg"], m[weights], prompt + done)[-1]
            z = ref_perturbed(under_rules(logits, sp, prompt, done, eng.stop_token_ids), sp.temperature, sp.seed or 0, i)
            # a logit that is off by d is off by d times 1 / repetition or repetition after the penalty
            stretch = max(sp.repetition_penalty, 1 / sp.repetition_penalty) / max(sp.temperature, 1e-9 if sp.temperature else 1.0)
            assert float(z.max() - z[tok]) <= slack_rel * float(logits.abs().max()) * stretch, f"output {i}: {tok}, plain {int(z.argmax())}"
            done.append(tok)


def even_then_small(output):
    """A little grammar: after an even token any multiple of three, after an odd one the first twenty, at the start anything."""
    if not output:
        return None
    return range(0, 240, 3) if output[-1] % 2 == 0 else range(20)


PARAMS = [dict(repetition_penalty=1.8), dict(frequency_penalty=0.7, presence_penalty=0.4, temperature=0.9, seed=3), dict(),
          dict(logit_bias={5: 3.0, 7: -math.inf, 100: 2.5}, presence_penalty=1.0), dict(temperature=0.8, seed=11),
          dict(repetition_penalty=0.7, frequency_penalty=-0.5)]


def run(m, device, dtype, slack, params, weights="weights", **cfg):
    prompts = prompts_for(m, [5, 17, 33, 1, 9, 26][:len(params)], seed=5)
    eng = engine(m, device, dtype, **{**dict(num_blocks=40, max_num_seqs=6, max_num_batched_tokens=32), **cfg})
    params = [SamplingParams(max_tokens=12, ignore_eos=True, **p) for p in params]
    outs = eng.generate(prompts, params)
    assert all(len(o.output_ids) == 12 for o in outs)
    check(m, eng, prompts, outs, params, slack, weights)
    eng.cache.check()
    return eng, [o.output_ids for o in outs]


@pytest.mark.parametrize("ahead", [True, False])
def test_rules_host(tiny_models, ahead):
    eng, tokens = run(tiny_models["A"], "cpu", "float32", 1e-6, PARAMS, run_ahead=ahead)
    # the rules changed something, and requests without any are as they would be alone
    _, free = run(tiny_models["A"], "cpu", "float32", 1e-6, [{k: v for k, v in p.items() if k in ("temperature", "seed")} for p in PARAMS])
    assert tokens[2] == free[2] and tokens[4] == free[4] and tokens[0] != free[0]


def test_a_step_ahead_changes_no_token_host(tiny_models):
    a = run(tiny_models["B"], "cpu", "float32", 1e-6, PARAMS, run_ahead=True)[1]
    assert a == run(tiny_models["B"], "cpu", "float32", 1e-6, PARAMS, run_ahead=False)[1]


def test_rules_under_preemption_host(tiny_models):
    m = tiny_models["A"]
    prompts = prompts_for(m, [30, 28, 33, 20], seed=2)
    params = [SamplingParams(max_tokens=24, ignore_eos=True, repetition_penalty=1.5, frequency_penalty=0.3)] * 4
    roomy = engine(m, "cpu", "float32", num_blocks=40, max_num_seqs=4).generate(prompts, params)
    tight = engine(m, "cpu", "float32", num_blocks=10, max_num_seqs=4)
    outs = tight.generate(prompts, params)
    assert tight.scheduler.num_preemptions > 0
    assert [o.output_ids for o in outs] == [o.output_ids for o in roomy]
    check(m, tight, prompts, outs, params, 1e-6)


def test_requests_without_rules_ask_for_nothing(tiny_models):
    eng, _ = run(tiny_models["A"], "cpu", "float32", 1e-6, [dict(), dict(temperature=0.5, seed=1)])
    assert eng.runner.token_history is None and "record_tokens" not in eng.runner.ops.calls
    assert "sample under rules" not in eng.runner.ops.calls


def test_allowed_tokens_host(tiny_models):
    calls = []

    def grammar(output):
        calls.append(len(output))
        assert -1 not in output                       # nothing that is still on its way
        return even_then_small(output)

    eng, tokens = run(tiny_models["A"], "cpu", "float32", 1e-6, [dict(allowed_tokens=grammar), dict(), dict(repetition_penalty=1.3)])
    assert set(calls) == set(range(12))
    for a, b in zip(tokens[0], tokens[0][1:]):
        assert b in even_then_small([a])
    _, free = run(tiny_models["A"], "cpu", "float32", 1e-6, [dict(), dict(), dict()])
    assert tokens[1] == free[1]
    assert not eng._reading and eng._in_flight is None


def test_allowed_tokens_beside_a_step_in_flight_host(tiny_models):
    """A request that reads its output joins while others run a step ahead, and leaves again."""
    m = tiny_models["A"]
    prompts = prompts_for(m, [9, 12, 7], seed=3)
    eng = engine(m, "cpu", "float32", num_blocks=40, max_num_seqs=4)
    long = SamplingParams(max_tokens=20, ignore_eos=True, presence_penalty=0.5)
    short = SamplingParams(max_tokens=5, ignore_eos=True, allowed_tokens=even_then_small)
    seqs = [eng.add_request(prompts[0], long)]
    done = []
    for i in range(60):
        if i == 4:
            seqs.append(eng.add_request(prompts[1], short))
        if i == 7:
            seqs.append(eng.add_request(prompts[2], long))
        if not eng.has_work():
            break
        done += eng.step()
    assert sorted(s.seq_id for s in done) == sorted(s.seq_id for s in seqs)
    for s, p in zip(seqs, (long, short, long)):
        assert len(s.output_ids) == p.max_tokens
        check(m, eng, [s.token_ids[:s.prompt_len]], [s], [p], 1e-6)


def test_where_nothing_is_allowed_the_request_ends(tiny_models):
    m = tiny_models["A"]
    eng = engine(m, "cpu", "float32", num_blocks=40)
    sp = SamplingParams(max_tokens=20, allowed_tokens=lambda out: range(10, 30) if len(out) < 3 else ())
    out = eng.generate(prompts_for(m, [6], seed=1), sp)[0].output_ids
    assert len(out) == 4 and out[-1] == m["cfg"]["eos_token_id"] and all(10 <= t < 30 for t in out[:3])
    eng.eos_token_id = None
    with pytest.raises(ValueError, match="no token is allowed"):
        eng.generate(prompts_for(m, [6], seed=1), sp)


def test_a_step_whose_rules_fail_can_be_taken_again(tiny_models):
    """allowed_tokens that raises once, and once gives what is no token: the step is not taken, and the same one follows."""
    m = tiny_models["A"]
    want = run(m, "cpu", "float32", 1e-6, [dict(allowed_tokens=even_then_small), dict(repetition_penalty=1.4), dict()])[1]
    calls = []

    def sometimes(output):
        calls.append(len(output))
        if len(calls) == 3:
            raise KeyError("not now")
        return [10 ** 6] if len(calls) == 6 else even_then_small(output)

    eng = engine(m, "cpu", "float32", num_blocks=40, max_num_seqs=6, max_num_batched_tokens=32)
    seqs = [eng.add_request(p, SamplingParams(max_tokens=12, ignore_eos=True, **sp)) for p, sp in
            zip(prompts_for(m, [5, 17, 33], seed=5), [dict(allowed_tokens=sometimes), dict(repetition_penalty=1.4), dict()])]
    failed = []
    while eng.has_work():
        try:
            eng.step()
        except (KeyError, ValueError) as e:
            failed.append(type(e))
        eng.cache.check()
    assert failed == [KeyError, ValueError] and len(calls) == 14
    assert [s.output_ids for s in seqs] == want


def test_a_refused_request_leaves_the_engine_as_it_was(tiny_models):
    eng = engine(tiny_models["A"], "cpu", "float32", num_blocks=4, max_num_seqs=2, max_num_batched_tokens=32)
    with pytest.raises(Exception, match="pages|blocks|tokens"):
        eng.add_request([1] * 200, SamplingParams(max_tokens=300, repetition_penalty=1.5, allowed_tokens=even_then_small))
    assert not eng.has_work() and not eng._reading


def test_mask_words():
    w = mask_words([0, 31, 32, 99], 100)
    assert w.tolist() == [1 | -2**31, 1, 0, 8]
    assert not mask_words([], 33).any() and len(mask_words([], 33)) == 2
    for bad in ([100], [-1]):
        with pytest.raises(ValueError, match="vocabulary"):
            mask_words(bad, 100)


@pytest.mark.parametrize("bad", [dict(repetition_penalty=0.0), dict(repetition_penalty=math.inf), dict(repetition_penalty=math.nan),
                                 dict(presence_penalty=math.nan), dict(frequency_penalty=math.inf), dict(logit_bias={1: math.nan}),
                                 dict(logit_bias={"a": 1.0}), dict(allowed_tokens=[1, 2])])
def test_refused_params(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad)


def test_biases_outside_the_vocabulary_are_refused(tiny_models):
    eng = engine(tiny_models["A"], "cpu", "float32", num_blocks=16)
    with pytest.raises(ValueError, match="vocabulary"):
        eng.add_request([1, 2], SamplingParams(logit_bias={256: 1.0}))
    assert not eng.has_work()


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("model", ["A", "C"])
def test_rules_gpu(tiny_models, model, graphs):
    params = PARAMS + [dict(allowed_tokens=even_then_small, temperature=0.7, seed=5)] if not graphs else PARAMS
    params = params[-6:]
    for dtype, slack, weights in (("float32", 1e-5, "weights"), ("bfloat16", 2e-2, "weights_bf16")):
        m = tiny_models[model]
        eng, tokens = run(m, "cuda", dtype, slack, params, weights, use_hip_graphs=graphs, graph_batch_sizes=(1, 2, 4, 6))
        assert (eng.num_graph_steps > 0) == graphs
        again = run(m, "cuda", dtype, slack, params, weights, use_hip_graphs=graphs, graph_batch_sizes=(1, 2, 4, 6), run_ahead=False)[1]
        assert tokens == again


@pytest.mark.gpu
def test_allowed_tokens_gpu(tiny_models):
    m = tiny_models["A"]
    eng, tokens = run(m, "cuda", "bfloat16", 2e-2, [dict(allowed_tokens=even_then_small), dict(), dict(repetition_penalty=1.3)], "weights_bf16",
                      graph_batch_sizes=(1, 2, 4))
    for a, b in zip(tokens[0], tokens[0][1:]):
        assert b in even_then_small([a])


@pytest.mark.gpu
def test_rules_under_preemption_gpu(tiny_models):
    m = tiny_models["A"]
    prompts = prompts_for(m, [30, 28, 33, 20], seed=2)
    params = [SamplingParams(max_tokens=24, ignore_eos=True, repetition_penalty=1.5, frequency_penalty=0.3)] * 4
    tight = engine(m, "cuda", "float32", num_blocks=10, max_num_seqs=4, graph_batch_sizes=(1, 2, 4))
    outs = tight.generate(prompts, params)
    assert tight.scheduler.num_preemptions > 0
    check(m, tight, prompts, outs, params, 1e-5)
