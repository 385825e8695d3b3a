"""Rules on logits (penalties, biases, masks) and the choice of tokens under them, against a plain implementation in 64 bits.

Tolerance: a logit passes at most five operations of 32 bits (division or product, product, two subtractions, addition), each off by
at most 2^-24 of its result; with |z| the largest magnitude met on the way the sum of the errors is at most 5 * 2^-24 * |z|.
"""
import dataclasses
import math
import sys

import pytest
import torch

from mini_inference_engine_amd.kernels.api import LogitRules
from mini_inference_engine_amd.kernels.hip_backend import HipBackend


def make(R, V, history, seed, dev, masked=True, biased=8):
    g = torch.Generator().manual_seed(seed)
    slots = R + 2
    ids = torch.randint(0, max(1, V // 3), (slots, history + 3), generator=g)
    lengths = torch.randint(0, history + 1, (R,), generator=g)
    lengths[0] = history
    prompt = (lengths * torch.rand(R, generator=g)).long()
    starts = torch.cumsum(torch.cat([torch.zeros(1, dtype=torch.long), torch.randint(0, biased + 1, (R,), generator=g)]), 0)
    N = int(starts[-1])
    words = (V + 31) // 32
    masks = torch.randint(-2**31, 2**31, (3, words + 1), generator=g)
    masks[1] = 0                     # nothing may come
    d = dict(history=ids, slots=torch.randperm(slots, generator=g)[:R], lengths=lengths, prompt_lengths=prompt,
             repetition=0.5 + 1.5 * torch.rand(R, generator=g), presence=torch.rand(R, generator=g) - 0.3,
             frequency=torch.rand(R, generator=g) - 0.2, bias_starts=starts, bias_tokens=torch.randint(0, V, (N,), generator=g),
             bias_values=4 * torch.randn(N, generator=g))
    if masked:
        d.update(masks=masks, mask_rows=torch.randint(-1, 3, (R,), generator=g))
    if R > 1:
        d["repetition"][1], d["presence"][1], d["frequency"][1] = 1.0, 0.0, 0.0
    f = ("repetition", "presence", "frequency", "bias_values")
    return LogitRules(**{k: (v.float() if k in f else v.to(torch.int32)).to(dev) for k, v in d.items()})


def plain(logits, rules):
    """-> adjusted logits in 64 bits, and the largest magnitude met on the way."""
    z = logits.double().cpu().clone()
    R, V = z.shape
    most = torch.nan_to_num(z.abs(), nan=0.0)
    c = {k: (None if v is None else v.cpu()) for k, v in vars(rules).items()}
    for r in range(R):
        if c["history"] is not None and 0 <= int(c["slots"][r]) < c["history"].shape[0]:
            n = max(0, min(int(c["lengths"][r]), c["history"].shape[1]))
            text = c["history"][int(c["slots"][r]), :n].tolist()
            rep, fre, pre = float(c["repetition"][r]), float(c["frequency"][r]), float(c["presence"][r])
            for v in sorted(set(text)):
                if not 0 <= v < V:
                    continue
                z[r, v] = z[r, v] / rep if z[r, v] > 0 else z[r, v] * rep
                most[r, v] = max(most[r, v], abs(z[r, v]))
                k = text[int(c["prompt_lengths"][r]):].count(v)
                if k:
                    most[r, v] += abs(fre * k) + abs(pre)
                    z[r, v] -= fre * k + pre
        if c["bias_starts"] is not None:
            last = {}
            for i in range(int(c["bias_starts"][r]), int(c["bias_starts"][r + 1])):
                last[int(c["bias_tokens"][i])] = float(c["bias_values"][i])
            for v, b in last.items():
                if 0 <= v < V:
                    most[r, v] += abs(b)
                    z[r, v] += b
        if c["masks"] is not None and 0 <= int(c["mask_rows"][r]) < c["masks"].shape[0]:
            bits = (c["masks"][int(c["mask_rows"][r])].long()[:, None] >> torch.arange(32)) & 1
            z[r, bits.reshape(-1)[:V] == 0] = -math.inf
    return z, most


def check_adjusted(got, want, most):
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    assert ((got - want).abs()[fine] <= 5 * 2.0 ** -24 * most[fine]).all()


@pytest.fixture(scope="module")
def ops():
    return HipBackend(torch.bfloat16)


SIZES = [(1, 1, 1), (1, 5, 3), (3, 31, 40), (2, 1023, 17), (5, 1024, 300), (4, 1025, 1), (2, 4099, 2000), (7, 50261, 700), (1, 128256, 5000),
         (130, 33000, 100), (300, 20001, 257), (9, 8192, 50), (9, 8193, 50), (3, 12289, 4000)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES)
def test_adjusted_logits(ops, size):
    R, V, history = size
    rules = make(R, V, history, 5, "cuda")
    logits = 4 * torch.randn((R, V), generator=torch.Generator().manual_seed(1))
    logits[0, V // 2] = math.inf
    logits[R - 1, V // 3] = -math.inf
    if R > 2:
        logits[2, ::7] = math.nan
    logits = logits.cuda()
    kept = logits.clone()
    want, most = plain(logits, rules)
    got = ops.adjust_logits(logits, rules)
    assert torch.equal(logits.nan_to_num(nan=7.0), kept.nan_to_num(nan=7.0))
    check_adjusted(got, want, most)
    # in place, and twice the same bits
    again = ops.adjust_logits(kept, rules, out=kept)
    assert again is kept and torch.equal(again.view(torch.int32), got.view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1029, 20005])
@pytest.mark.parametrize("offset, stride", [(0, 2), (1, 3), (3, 7), (4, 7)])
def test_adjusted_logits_of_rows_anywhere(ops, V, offset, stride):
    R, stride = 5, V + stride
    rules = make(R, V, 60, 9, "cuda")
    pool = torch.randn(R * stride + 8, generator=torch.Generator().manual_seed(2)).cuda()
    logits = pool[offset:offset + R * stride].view(R, stride)[:, :V]
    out_pool = torch.full((R * stride + 8,), 77.0, device="cuda")
    out = out_pool[offset:offset + R * stride].view(R, stride)[:, :V]
    want, most = plain(logits, rules)
    check_adjusted(ops.adjust_logits(logits, rules, out=out), want, most)
    temps, seeds, counters = torch.zeros(R, device="cuda"), torch.zeros(R, dtype=torch.int64, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.sample(logits, temps, seeds, counters, rules=rules), ops.sample(out, temps, seeds, counters))
    mine = torch.zeros(R * stride + 8, dtype=torch.bool, device="cuda")
    mine[offset:offset + R * stride].view(R, stride)[:, :V] = True
    assert (out_pool[~mine] == 77.0).all()          # nothing beside the rows is written


@pytest.mark.gpu
@pytest.mark.parametrize("group", ["penalties", "biases", "masks", "none"])
def test_each_group_of_rules_alone(ops, group):
    R, V = 6, 3001
    names = {"penalties": ("history", "slots", "lengths", "prompt_lengths", "repetition", "presence", "frequency"),
             "biases": ("bias_starts", "bias_tokens", "bias_values"), "masks": ("masks", "mask_rows"), "none": ()}[group]
    full = make(R, V, 90, 3, "cuda")
    rules = LogitRules(**{n: getattr(full, n) for n in names})
    logits = torch.randn((R, V), generator=torch.Generator().manual_seed(4)).cuda()
    want, most = plain(logits, rules)
    check_adjusted(ops.adjust_logits(logits, rules), want, most)
    temps, seeds, counters = torch.zeros(R, device="cuda"), torch.zeros(R, dtype=torch.int64, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
    chosen = ops.sample(logits, temps, seeds, counters, rules=rules)
    assert torch.equal(chosen, ops.sample(ops.adjust_logits(logits, rules), temps, seeds, counters))
    if group == "none":
        assert torch.equal(chosen, ops.sample(logits, temps, seeds, counters))


@pytest.mark.gpu
def test_what_is_out_of_range_counts_for_nothing(ops):
    """Tokens outside the vocabulary in a text or a list, slots outside the history, lengths beyond it, mask rows that are none."""
    R, V = 6, 500
    rules = make(R, V, 40, 11, "cuda")
    rules.history[:, ::3] = V
    rules.history[:, 1::5] = -1
    rules.history[:, 2::7] = 2**31 - 1
    rules.slots[2], rules.slots[3] = -1, 10**6
    rules.lengths[4] = 43                            # all of the history's positions
    rules.mask_rows[5], rules.mask_rows[0] = 3, -7
    rules.bias_tokens[0], rules.bias_tokens[1] = V, -1
    logits = torch.randn((R, V), generator=torch.Generator().manual_seed(4)).cuda()
    want, most = plain(logits, rules)
    check_adjusted(ops.adjust_logits(logits, rules), want, most)
    rules.lengths[4] = 2**31 - 1                     # more than there are: those that are there
    check_adjusted(ops.adjust_logits(logits, rules), want, most)


@pytest.mark.gpu
def test_the_last_of_a_tokens_biases_counts(ops):
    V = 2000
    starts = torch.tensor([0, 500, 500, 502], dtype=torch.int32, device="cuda")
    tokens = torch.tensor([7] * 400 + [1999] * 100 + [3, 3], dtype=torch.int32, device="cuda")
    values = torch.arange(502, dtype=torch.float32, device="cuda")
    out = ops.adjust_logits(torch.zeros((3, V), device="cuda"), LogitRules(bias_starts=starts, bias_tokens=tokens, bias_values=values))
    want = torch.zeros((3, V))
    want[0, 7], want[0, 1999], want[2, 3] = 399, 499, 501
    assert torch.equal(out.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES)
def test_choice_under_rules_is_the_choice_from_adjusted_logits(ops, size):
    R, V, history = size
    rules = make(R, V, history, 6, "cuda")
    g = torch.Generator().manual_seed(8)
    logits = (4 * torch.randn((R, V), generator=g)).round(decimals=1)         # many equals
    logits[R - 1, V // 4] = math.nan
    logits = logits.cuda()
    temps = torch.where(torch.arange(R) % 2 == 0, torch.zeros(R), torch.rand(R, generator=g) + 0.3).cuda()
    seeds = torch.randint(-2**62, 2**62, (R,), generator=g).cuda()
    counters = torch.randint(0, 1000, (R,), generator=g).to(torch.int32).cuda()
    adjusted = ops.adjust_logits(logits, rules)
    want = ops.sample(adjusted, temps, seeds, counters)
    out = torch.full((R,), -5, dtype=torch.int32, device="cuda")
    got = ops.sample(logits, temps, seeds, counters, out=out, rules=rules)
    assert got is out and torch.equal(got, want)
    # greedy rows from the definition
    z, _ = plain(logits, rules)
    for r in range(0, R, 2):
        z32 = torch.nan_to_num(adjusted[r].cpu(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        assert int(got[r]) == int((z32 == z32.max()).nonzero()[0, 0])
        if torch.isinf(z[r]).all():
            assert int(got[r]) == 0


@pytest.mark.gpu
def test_choice_under_rules_in_a_graph_and_on_another_stream(ops):
    R, V = 9, 32000
    rules = make(R, V, 200, 21, "cuda")
    logits = torch.randn((R, V), device="cuda")
    temps, seeds = torch.full((R,), 0.7, device="cuda"), torch.arange(R, device="cuda")
    counters = torch.zeros(R, dtype=torch.int32, device="cuda")
    out, adjusted = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros_like(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample(logits, temps, seeds, counters, out=out, rules=rules)
        ops.adjust_logits(logits, rules, out=adjusted)
    torch.cuda.synchronize()
    assert torch.equal(out, ops.sample(adjusted, temps, seeds, counters))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adjust_logits(logits, rules, out=adjusted)
        ops.sample(logits, temps, seeds, counters, out=out, rules=rules)
    for i in range(4):
        logits.copy_(torch.randn((R, V), generator=torch.Generator().manual_seed(i)))
        counters.fill_(i)
        rules.lengths.fill_(20 * i)
        rules.prompt_lengths.fill_(10 * i)
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.adjust_logits(logits, rules)
        assert torch.equal(adjusted, eager)
        assert torch.equal(out, ops.sample(eager, temps, seeds, counters))


class Step:
    taken_from = earlier_tokens = None


def recorded(history, step):
    want = history.clone()
    for t in range(step.num_tokens):
        r, p = int(step.token_row[t]), int(step.positions[t])
        s = int(step.state_slots[r])
        tok = int(step.input_ids[t])
        if step.taken_from is not None and int(step.taken_from[t]) >= 0:
            tok = int(step.earlier_tokens[int(step.taken_from[t])])
        if 0 <= s < history.shape[0] and 0 <= p < history.shape[1]:
            want[s, p] = tok
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("T, rows", [(1, 1), (300, 7), (256, 256), (1500, 3)])
@pytest.mark.parametrize("taken", [False, True])
def test_recorded_tokens(ops, T, rows, taken):
    g = torch.Generator().manual_seed(T)
    s = Step()
    s.num_tokens, s.num_rows = T, rows
    s.token_row = torch.sort(torch.randint(0, rows, (T,), generator=g)).values.to(torch.int32)
    s.positions = torch.arange(T, dtype=torch.int32) - 2            # two before the first, some beyond the last
    s.input_ids = torch.randint(0, 1000, (T,), generator=g).to(torch.int32)
    s.state_slots = (torch.randperm(rows, generator=g) + 1).to(torch.int32)     # one of them outside
    if taken:
        s.taken_from = torch.where(torch.rand(T, generator=g) < 0.5, torch.randint(0, 20, (T,), generator=g), -torch.ones(T, dtype=torch.long)).to(torch.int32)
        s.earlier_tokens = torch.randint(0, 1000, (20,), generator=g).to(torch.int32)
    pool = torch.full((rows, max(1, T - 5) + 3), -9, dtype=torch.int32)
    want = recorded(pool[:, :max(1, T - 5)], s)
    for name in ("token_row", "positions", "input_ids", "state_slots", "taken_from", "earlier_tokens"):
        if getattr(s, name) is not None:
            setattr(s, name, getattr(s, name).cuda())
    dev = pool.cuda()
    ops.record_tokens(dev[:, :max(1, T - 5)], s)
    assert torch.equal(dev[:, :max(1, T - 5)].cpu(), want)
    assert (dev[:, max(1, T - 5):] == -9).all()


# ---- refusals, on the CPU: the checks are made before anything is launched (a CPU tensor's device index is -1)

@pytest.fixture
def checks():
    b = object.__new__(HipBackend)
    b._device_index = -1
    return b


BAD = [("slots", lambda t: t.long()), ("slots", lambda t: t[:-1]), ("lengths", lambda t: None), ("prompt_lengths", lambda t: t.float()),
       ("repetition", lambda t: t.double()), ("presence", lambda t: t[None]), ("frequency", lambda t: torch.stack([t, t], 1)[:, 0]),
       ("history", lambda t: t.t()), ("history", lambda t: t.long()), ("history", lambda t: t[0]), ("history", lambda t: t[:1].expand(4, -1)),
       ("bias_starts", lambda t: t[:-1]), ("bias_values", lambda t: t[:-1]), ("bias_tokens", lambda t: t.long()), ("bias_tokens", lambda t: None),
       ("masks", lambda t: t[:, :-2]), ("masks", lambda t: t.bool()), ("mask_rows", lambda t: None), ("mask_rows", lambda t: t.long())]


@pytest.mark.parametrize("bad", range(len(BAD)))
def test_refused_rules(checks, bad):
    R, V = 4, 100
    rules = make(R, V, 10, 0, "cpu")
    assert len(checks._rules_arguments("sample", rules, R, V)) == 18
    name, spoil = BAD[bad]
    setattr(rules, name, spoil(getattr(rules, name)))
    with pytest.raises(ValueError, match=name):
        checks._rules_arguments("sample", rules, R, V)


def test_rules_on_another_device_are_refused(checks):
    rules = make(2, 50, 4, 0, "cpu")
    checks._device_index = 0
    with pytest.raises(ValueError, match="this GPU"):
        checks._rules_arguments("sample", rules, 2, 50)


@pytest.mark.gpu
def test_refused_results(ops):
    logits = torch.zeros((2, 64), device="cuda")
    none = LogitRules()
    with pytest.raises(ValueError, match="out"):
        ops.adjust_logits(logits, none, out=torch.zeros((2, 64), device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="out"):
        ops.adjust_logits(logits, none, out=torch.zeros((2, 32), device="cuda"))
    with pytest.raises(ValueError, match="apart"):
        pool = torch.zeros(300, device="cuda")
        ops.adjust_logits(pool[:128].view(2, 64), none, out=pool[4:132].view(2, 64))
    with pytest.raises(ValueError, match="logits"):
        ops.adjust_logits(logits.double(), none)
    assert ops.adjust_logits(logits[:0], none).shape == (0, 64)
    nobody = torch.zeros(0, device="cuda")
    for V in (64, 50000):
        assert ops.sample(torch.zeros((0, V), device="cuda"), nobody, nobody.long(), nobody.to(torch.int32), rules=none).shape == (0,)
    wide = torch.zeros((1, 64), device="cuda").expand(2, 64)          # rows on top of one another
    with pytest.raises((ValueError, RuntimeError), match="logits|leading"):
        ops.adjust_logits(wide, none, out=torch.zeros((2, 64), device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("R, V", [(7, 50261), (300, 20001), (64, 128256)])
def test_calls_one_after_another_and_on_two_streams(ops, R, V):
    """The last workgroup of a row joins the row's slices, by counters that every call leaves as it found them: many calls, sizes that
    change in between, two streams at once, against the choice from adjusted logits."""
    rules = make(R, V, 50, 4, "cuda")
    temps, seeds = torch.zeros(R, device="cuda"), torch.arange(R, device="cuda")
    counters = torch.zeros(R, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    inputs = [torch.randn((R, V), generator=g, device="cuda") for _ in range(4)]
    wants = [ops.sample(ops.adjust_logits(x, rules), temps, seeds, counters) for x in inputs]
    small = make(3, 33000, 5, 9, "cuda")
    x_small = torch.randn((3, 33000), generator=g, device="cuda")
    want_small = ops.sample(ops.adjust_logits(x_small, small), temps[:3], seeds[:3], counters[:3])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 4, ops.sample(inputs[i % 4], temps, seeds, counters, rules=rules)))
            if i % 5 == 0:
                got.append((-1, ops.sample(x_small, temps[:3], seeds[:3], counters[:3], rules=small)))
    torch.cuda.synchronize()
    for i, t in got:
        assert torch.equal(t, want_small if i < 0 else wants[i])


@pytest.mark.gpu
def test_a_captured_choice_beside_calls(ops):
    """Replays of two graphs on two streams beside calls on a third: each has memory of its own."""
    R, V = 40, 40000
    rules = make(R, V, 50, 4, "cuda")
    temps, seeds = torch.zeros(R, device="cuda"), torch.arange(R, device="cuda")
    counters = torch.zeros(R, dtype=torch.int32, device="cuda")
    inputs = [torch.randn((R, V), generator=torch.Generator().manual_seed(i)).cuda() for i in range(3)]
    wants = [ops.sample(ops.adjust_logits(x, rules), temps, seeds, counters) for x in inputs]
    outs = [torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(2)]
    graphs = []
    for x, out in zip(inputs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.sample(x, temps, seeds, counters, out=out, rules=rules)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        with torch.cuda.stream(streams[2]):
            here = [ops.sample(inputs[2], temps, seeds, counters, rules=rules) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1]) and all(torch.equal(h, wants[2]) for h in here)


class TheLongWay:
    """Declines every call, as the short way declines what it does not take."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def long_ops(ops):
    ops.adjust_logits(torch.zeros((1, 8), device="cuda"), LogitRules())          # (the short way is there)
    short, ops._direct = ops._direct, TheLongWay()
    yield ops
    ops._direct = short


def calls(ops, size, out):
    R, V, history = size
    rules = make(R, V, history, 11, "cuda")
    g = torch.Generator().manual_seed(4)
    logits = 4 * torch.randn((R, V + 5), generator=g).cuda()[:, :V]
    temps, seeds, counters = torch.rand(R, generator=g).cuda(), torch.arange(R).cuda() * 7919, torch.arange(R, dtype=torch.int32).cuda()
    made = []
    for _ in range(2):                              # (the first choice on a stream makes its workspace, and goes the long way)
        chosen = torch.full((R,), -5, dtype=torch.int32, device="cuda") if out else None
        adjusted = torch.full((R, V + 3), 9.0, device="cuda")[:, :V] if out else None
        made += [ops.sample(logits, temps, seeds, counters, out=chosen, rules=rules), ops.adjust_logits(logits, rules, out=adjusted)]
        assert not out or (made[-2] is chosen and made[-1] is adjusted)
    return made


@pytest.mark.gpu
@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("size", SIZES[:9])
def test_both_ways_into_the_kernels(ops, size, out):
    made = calls(ops, size, out)
    short, ops._direct = ops._direct, TheLongWay()
    try:
        for a, b in zip(made, calls(ops, size, out)):
            assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(torch.int32), b.view(torch.int32))
    finally:
        ops._direct = short


@pytest.mark.gpu
def test_a_call_keeps_nothing(ops):
    """References to what a call was given are as before, taken or declined, and so is the memory."""
    R, V = 5, 20001
    rules = make(R, V, 40, 3, "cuda")
    logits, out = torch.randn((R, V), device="cuda"), torch.empty((R, V), device="cuda")
    temps, seeds, counters = torch.ones(R, device="cuda"), torch.arange(R).cuda(), torch.zeros(R, dtype=torch.int32, device="cuda")
    held = [logits, out, temps, seeds, counters, rules, rules.history, rules.slots, rules.masks, rules.bias_values, None]

    def some():
        for _ in range(50):
            ops.sample(logits, temps, seeds, counters, rules=rules)
            ops.adjust_logits(logits, rules, out=out)
            ops.adjust_logits(logits, rules)
            for bad in (dict(seeds=counters), dict(logits=logits.double()), dict(temperatures=None), dict(rules=None)):
                kw = {**dict(logits=logits, temperatures=temps, seeds=seeds, counters=counters, rules=rules), **bad}
                if kw["rules"] is None:
                    with pytest.raises(AttributeError):
                        ops.adjust_logits(logits, None)
                else:
                    with pytest.raises(ValueError):
                        ops.sample(**kw)

    some()
    torch.cuda.synchronize()
    before, memory = [sys.getrefcount(x) for x in held[:-1]], torch.cuda.memory_allocated()
    some()
    torch.cuda.synchronize()
    assert [sys.getrefcount(x) for x in held[:-1]] == before and torch.cuda.memory_allocated() == memory


@pytest.mark.gpu
@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("name, change", [
    ("slots", lambda t: t.long()), ("lengths", lambda t: t[:-1]), ("prompt_lengths", lambda t: t.cpu()), ("repetition", lambda t: t.double()),
    ("presence", lambda t: torch.stack([t, t], 1)[:, 0]), ("frequency", lambda t: None), ("history", lambda t: t.long()), ("history", lambda t: t[0]),
    ("history", lambda t: t[:1].expand(3, -1)), ("bias_starts", lambda t: t[:-1]), ("bias_tokens", lambda t: t[:-1]), ("bias_values", lambda t: t.half()),
    ("masks", lambda t: t[:, :-2]), ("masks", lambda t: t.cpu()), ("mask_rows", lambda t: t[None])])
def test_refusals_of_both_ways(ops, long_ops, name, change, short):
    R, V = 4, 10007
    rules = make(R, V, 40, 3, "cuda")
    logits = torch.randn((R, V), device="cuda")
    small = torch.ones(R, device="cuda"), torch.arange(R).cuda(), torch.zeros(R, dtype=torch.int32, device="cuda")
    if short:
        ops._direct = ops.lib("direct_calls")
    ops.sample(logits, *small, rules=rules)
    bad = dataclasses.replace(rules, **{name: change(getattr(rules, name))})
    for call in (lambda: ops.sample(logits, *small, rules=bad), lambda: ops.adjust_logits(logits, bad)):
        with pytest.raises(ValueError, match="bias_values" if name == "bias_tokens" else name):      # (as many values as tokens)
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 70, 4099, 8192, 20001, 33000])
@pytest.mark.parametrize("hot", [0.0, 0.7])
def test_equals_and_rows_without_numbers(ops, V, hot):
    """The lowest index among equals, wherever its thread, wave or slice; of a row of -infinity and NaN the first -infinity; of NaN alone 0."""
    g = torch.Generator().manual_seed(V)
    R = 12
    logits = torch.randint(-2, 3, (R, V), generator=g).float()
    logits[1] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    logits[2] = -math.inf
    logits[3], logits[4] = math.nan, math.nan
    logits[4, V * 2 // 3:] = -math.inf
    logits[5, :V - 1] = math.nan
    logits[6] = 1.0
    logits[7, ::2] = math.inf
    logits[8] = 3.0
    rules = make(R, V, 60, 3, "cuda", masked=False)
    for name, value in (("repetition", 1.0), ("presence", 0.0), ("frequency", 0.0)):
        getattr(rules, name)[:9] = value            # (the others' penalties and biases are whole numbers: equals remain)
        getattr(rules, name)[9:] = {"repetition": 2.0, "presence": 1.0, "frequency": 1.0}[name]
    rules.bias_values = rules.bias_values.round()
    starts = rules.bias_starts.clone()
    starts[:6] = 0
    rules.bias_starts = starts
    masks = torch.full((2, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    masks[1] = 0
    masks[1, -1] = 1
    rules.masks, rules.mask_rows = masks, torch.tensor([-1, -1, -1, -1, -1, -1, 0, 0, 1, 0, -1, -1], dtype=torch.int32, device="cuda")
    logits = logits.cuda()
    small = torch.full((R,), hot, device="cuda"), torch.arange(R).cuda() * 31, torch.arange(R, dtype=torch.int32).cuda()
    got = ops.sample(logits, *small, rules=rules)
    adjusted = ops.adjust_logits(logits, rules)
    assert torch.equal(got, ops.sample(adjusted, *small))
    if hot == 0:
        z = adjusted.cpu().nan_to_num(nan=-math.inf, neginf=-1e38)          # (-infinity above NaN)
        want = [int((row == row.max()).nonzero()[0]) if not torch.isnan(a).all() else 0 for row, a in zip(z, adjusted.cpu())]
        assert got.tolist() == want
