"""Steps given ``shared_prefix`` through the designs whose layers of full attention are parts.SoftmaxAttention (sinks for all heads or one a
head, values mixed or taken from keys), beside windows and state of fixed size: requests of such models share no pages (each is a run of its
own), and their steps are what they are without ``shared_prefix``, kernel by kernel and captured.

Tolerance: against the plain implementation in float32 as in the designs' own tests; in bfloat16 both steps are within a layer's
rounding times the layers of it, so within twice that of each other.
"""
import functools
import importlib

import pytest
import torch

from test_shared_answers import SharedBackend

from mini_inference_engine_amd.engine.batch import StepRow
from mini_inference_engine_amd.engine.runner import ModelRunner

DESIGNS = [("vezodra", "A"), ("vezodra", "B"), ("vezodra", "C"), ("pokulorn", "A"), ("pokulorn", "B"), ("pokulorn", "C"), ("bulitar", "B")]
LENGTHS = (5, 33, 60, 1)
STEPS = 4


def steps(name, design, device, dtype, shared, graphs=False, share=None):
    """Logits of every step, [steps][rows], the texts, and how many of the steps were captured."""
    mod = importlib.import_module("test_" + name)
    raw, cfg, weights = mod.make(design, torch.float32 if dtype == "float32" else torch.bfloat16, sharp=dtype == "float32")
    kw = dict(weights=weights, dtype=dtype, device=device, num_pages=64, max_rows=8, max_step_tokens=256, max_model_len=300)
    runner = ModelRunner(cfg, **kw, **({"backend": SharedBackend(torch.float32)} if device == "cpu" else {}))
    if graphs:
        runner.capture_decode_graphs((4, 8))
    if share is not None:
        runner.ops.plan_shared_prefix = functools.partial(runner.ops.plan_shared_prefix, share=share)
    g = torch.Generator().manual_seed(9)
    texts = [torch.randint(0, raw["vocab"], (n + STEPS,), generator=g).tolist() for n in LENGTHS]
    caches, got, captured = [], [], 0
    for i, n in enumerate(LENGTHS):
        rc = runner.cache.open(i)
        assert runner.cache.reserve(rc, 0, n + STEPS)
        runner.forward_step([StepRow(rc, texts[i][:n], 0)])
        caches.append(rc)
    for k in range(STEPS):
        rows = [StepRow(rc, [t[n + k]], n + k, [0]) for rc, t, n in zip(caches, texts, LENGTHS)]
        logits = runner.forward_step(rows, shared_prefix=[(1, 0)] * len(rows) if shared else None)
        captured += runner.last_step_captured
        got.append(logits.clone().double().cpu())
    return got, texts, captured, (mod, raw, weights, runner)


def check_plain(got, texts, mod, raw, weights):
    expected = mod.expected_logits(raw, weights, dict(enumerate(texts)))
    for k, logits in enumerate(got):
        for i, n in enumerate(LENGTHS):
            want = expected[i][n + k]
            assert float((logits[i] - want.double()).abs().max()) <= mod.F32_TOL * float(expected[i].abs().max()), (i, k)


@pytest.mark.parametrize("name, design", DESIGNS)
def test_designs_host(name, design):
    got, texts, _, (mod, raw, weights, runner) = steps(name, design, "cpu", "float32", True)
    assert runner.ops.calls["shared"] > 0
    check_plain(got, texts, mod, raw, weights)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs, share", [(False, True), (False, False), (True, True), (True, None)])
@pytest.mark.parametrize("name, design", DESIGNS)
def test_designs_gpu(name, design, graphs, share):
    got, texts, captured, (mod, raw, weights, _) = steps(name, design, "cuda", "float32", True, graphs, share)
    assert captured == (STEPS - 1 if graphs else 0)
    check_plain(got, texts, mod, raw, weights)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name, design", DESIGNS)
def test_designs_in_bfloat16(name, design, graphs):
    got, _, captured, (mod, raw, _, _) = steps(name, design, "cuda", "bfloat16", True, graphs, True)
    want = steps(name, design, "cuda", "bfloat16", False)[0]
    assert captured == (STEPS - 1 if graphs else 0)
    tol = 2 * mod.BF16_TOL_PER_LAYER * (mod.layer_runs(raw) if hasattr(mod, "layer_runs") else len(raw["layers"]))
    errs = [float((a - b).abs().max()) / float(b.abs().max()) for x, y in zip(got, want) for a, b in zip(x, y)]
    # (a router's near tie may choose another expert in some rows, as the designs' own tests allow)
    assert all(e <= 1.0 for e in errs) and sum(e > tol for e in errs) <= 0.25 * len(errs), sorted(errs)[-6:]
