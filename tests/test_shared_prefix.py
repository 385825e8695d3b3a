"""Attention of rows that share the first part of their cache, against a plain softmax in 64 bits over every row's own keys.

Tolerance.  out = sum p v / sum p with p = 2^(x - m).  With A = sum p |v| / sum p:  a score's error, relative to p, is
e = ln 2 * |error of x| + the exponential's: x = log2(e) scale q.k from 32-bit sums of D products, at most (D + 8) 2^-24 log2(e) scale
sum |q k|, and 2^-21 for the exponential, its argument's rounding (|x| up to 64) and the joins; p's sum of N terms adds N 2^-24.
Numerator and denominator both carry that: 2 (e + N 2^-24) A.  In bfloat16 the p of the numerator are rounded (2^-8 A) and the result is
(2^-8 |out|).
"""
import copy
import math
import pickle
import sys
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from mini_inference_engine_amd.kernels.hip_backend import HipBackend
from mini_inference_engine_amd.kernels.shared_prefix import SharedPrefixPlan, _sharers

BF16, F32 = torch.bfloat16, torch.float32


def make(groups, positions, Hq, Hkv, D, page, dtype, seed=0, poison=True, device="cuda", extra_stride=0, extra_pages=3):
    """``groups``: (rows, shared keys); ``positions`` of all rows.  -> what a step has, on the device."""
    g = torch.Generator().manual_seed(seed)
    T = len(positions)
    blocks = max(positions) // page + 1 + 2
    tables, used, at = torch.zeros((T, blocks), dtype=torch.int64), [], 1
    row = 0
    for n, keys in groups:
        whole = keys // page
        shared = torch.arange(at, at + whole)
        at += whole
        for r in range(row, row + n):
            need = max(0, positions[r] // page + 1 - whole) if positions[r] >= 0 else 0
            tables[r, :whole] = shared
            tables[r, whole:whole + need] = torch.arange(at, at + need)
            at += need
        row += n
    pages = at + extra_pages
    ids = torch.cat([torch.zeros(1, dtype=torch.long), torch.randperm(pages - 1, generator=g) + 1])
    tables = ids[tables]
    k = torch.randn((pages, Hkv, page, D), generator=g)
    v = torch.randn((pages, Hkv, D, page), generator=g) + 0.5
    row = 0
    for n, keys in groups:                   # the page in which the shared keys end: a copy a row
        w, rest = keys // page, keys % page
        for r in range(row + 1, row + n):
            if rest:
                k[tables[r, w], :, :rest] = k[tables[row, w], :, :rest]
                v[tables[r, w], :, :, :rest] = v[tables[row, w], :, :, :rest]
        row += n
    if poison:                               # slots that hold no key of anybody: NaN, which must not reach a result
        written = torch.zeros((pages, page), dtype=torch.bool)
        for r, p in enumerate(positions):
            for j in range(p + 1):
                written[tables[r, j // page], j % page] = True
        k.masked_fill_(~written[:, None, :, None], math.nan)
        v.masked_fill_(~written[:, None, None, :], math.nan)
    q = 1.5 * torch.randn((T, Hq * D + extra_stride), generator=g)
    t = dict(q=q.to(dtype), k=k.to(dtype), v=v.to(dtype), tables=tables.to(torch.int32), positions=torch.tensor(positions, dtype=torch.int32))
    t = {n: x.to(device) for n, x in t.items()}
    return SimpleNamespace(**t, T=T, page=page, blocks=blocks)


def step_of(s, most=None, **kw):
    ramp = torch.arange(s.T + 1, dtype=torch.int32, device=s.q.device)
    ends = s.positions.cpu().numpy().astype(np.int64) + 1
    d = dict(num_rows=s.T, num_decode_rows=s.T, num_tokens=s.T, token_row=ramp[:s.T], positions=s.positions,
             max_context=int(max(1, ends.max())) if most is None else most, host={"row_context": ends})
    d.update(kw)
    return SimpleNamespace(**d), SimpleNamespace(block_tables=s.tables)


def plain(s, Hq, Hkv, D, scale, sink=None):
    """-> result, tolerance base A, score magnitude, keys; 64 bits, row by row."""
    outs, As, mags = [], [], []
    k, v, q = s.k.double().cpu(), s.v.double().cpu(), s.q.double().cpu()
    for r, p in enumerate(s.positions.tolist()):
        if p < 0:
            outs.append(torch.zeros(Hq * D, dtype=torch.float64)); As.append(torch.zeros(Hq * D, dtype=torch.float64)); mags.append(0.0)
            continue
        pages = s.tables[r, :p // s.page + 1].long().cpu()
        kk = k[pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :p + 1]
        vv = v[pages].permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :p + 1]
        qq = q[r, :Hq * D].view(Hkv, Hq // Hkv, D)
        x = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
        mags.append(float((torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()) * scale).max()))
        if sink is not None:
            sk = torch.as_tensor(sink, dtype=torch.float64).cpu().expand(Hq).view(Hkv, Hq // Hkv, 1)
            w = torch.softmax(torch.cat([x, sk], -1), -1)[..., :-1]
        else:
            w = torch.softmax(x, -1)
        outs.append(torch.matmul(w, vv).reshape(-1))
        As.append(torch.matmul(w, vv.abs()).reshape(-1))
    return torch.stack(outs), torch.stack(As), max(mags), int(s.positions.max()) + 1


def check(got, want, A, mag, N, D, dtype):
    e = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -21 + N * 2.0 ** -24
    tol = 2 * e * A + 2.0 ** -24 * want.abs()
    if dtype == BF16:
        tol = tol + 2.0 ** -8 * (A * (1 + 4 * e) + want.abs() * (1 + 2.0 ** -7))
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol + 1e-30
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / (tol + 1e-30)).max()))


@pytest.fixture(scope="module")
def ops():
    return {BF16: HipBackend(BF16), F32: HipBackend(F32)}


def run(ops, s, groups, Hq, Hkv, D, dtype, scale=None, sink=None, contexts=None, **kw):
    """Shared, not shared, and as the plan chooses by itself."""
    scale = D ** -0.5 if scale is None else scale
    step, group = step_of(s, **kw)
    want = plain(s, Hq, Hkv, D, scale, sink)
    for share in (True, False, None):
        plan = ops[dtype].plan_shared_prefix(groups, [p + 1 for p in s.positions.tolist()] if contexts is None else contexts, Hq, Hkv, D, share=share)
        out = ops[dtype].shared_prefix_attention(s.q, Hq, Hkv, D, s.k, s.v, group, step, scale, plan, sink=sink)
        check(out, *want, D, dtype)
    return out, plan


def rows_behind(groups, own, seed=0):
    """Positions: every row has between 0 and ``own`` keys behind its shared ones, and at least one key."""
    g = np.random.RandomState(seed)
    return [max(0, keys + int(g.randint(0, own + 1)) - 1) for n, keys in groups for _ in range(n)]


GROUPS = [([(1, 0)], 1), ([(1, 5)], 3), ([(2, 1)], 1), ([(3, 16)], 20), ([(4, 200)], 40), ([(5, 31), (1, 0), (2, 33)], 70), ([(2, 0), (3, 64)], 40),
          ([(17, 700)], 90), ([(8, 96), (8, 97), (1, 300), (6, 1500)], 300), ([(40, 333)], 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(2, 1, 16), (3, 3, 32), (4, 2, 48), (32, 4, 64), (5, 1, 80), (6, 2, 96), (8, 2, 128), (20, 1, 64), (2, 2, 256), (8, 1, 256)])
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_shared_prefix_attention(ops, case, heads, dtype):
    groups, own = GROUPS[case]
    s = make(groups, rows_behind(groups, own, case), *heads, 16, dtype, seed=case)
    run(ops, s, groups, *heads, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(2, 1, 16), (3, 3, 32), (4, 2, 48), (32, 4, 64), (6, 2, 96), (8, 2, 128), (16, 1, 128), (20, 1, 64), (2, 2, 256), (8, 1, 256)])
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_items_of_a_wave_and_of_more_columns(ops, case, heads, dtype):
    """Plans for a few compute units: short rows a wave each, and, for some hundred, items as short as they get."""
    groups, own = GROUPS[case]
    Hq, Hkv, D = heads
    s = make(groups, rows_behind(groups, own, case), *heads, 16, dtype, seed=case)
    contexts = [p + 1 for p in s.positions.tolist()]
    waves = _sharers(D, dtype == F32) if Hq // Hkv <= 16 else 0
    for nobody in (False, True):
        if nobody:                              # padding in between, and a row in the middle of its own keys
            s.positions[::3] = -1
            s.positions[-1] = max(0, int(s.positions[-1]) - 5) if int(s.positions[-1]) - 5 >= groups[-1][1] else int(s.positions[-1])
        step, group = step_of(s, most=max(contexts))
        want = plain(s, *heads, D ** -0.5, 0.3)
        for units in (1, 7, 600):
            for share in (True, False):
                plan = SharedPrefixPlan(groups, contexts, *heads, "cuda", units=units, float32=dtype == F32, share=share)
                if units == 1:
                    alone = sum(c <= Hq // Hkv for _, c, *_ in plan.items.view(-1, 8).tolist())
                    assert plan.num_items - plan.whole_items <= alone and (waves > 0 or plan.whole_items == plan.num_items)
                check(ops[dtype].shared_prefix_attention(s.q, *heads, s.k, s.v, group, step, D ** -0.5, plan, sink=0.3), *want, D, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 8, 64), (16, 4, 128), (4, 4, 256)])
def test_hundreds_of_short_rows(ops, heads, dtype):
    """More workgroups than there is room for: rows of 1 to 460 keys, whole and behind some shared ones, a wave each."""
    g = np.random.RandomState(1)
    for groups in ([(300, 0)], [(130, 48), (1, 0), (200, 16)]):
        positions = [k + int(x) - 1 for n, k in groups for x in g.choice([1, 2, 31, 32, 33, 100, 440], n)]
        s = make(groups, positions, *heads, 16, dtype, poison=False)
        out, plan = run(ops, s, groups, *heads, dtype)
        assert plan.num_items - plan.whole_items > 100


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [16, 32, 48, 128])
def test_pages_of_other_sizes(ops, page, dtype):
    groups = [(3, 130), (2, 95), (4, 144)]
    s = make(groups, rows_behind(groups, 60, page), 8, 2, 64, page, dtype, seed=page)
    run(ops, s, groups, 8, 2, 64, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra", [1, 3, 8, 130])
def test_queries_of_any_stride(ops, extra, dtype):
    groups = [(5, 70)]
    s = make(groups, rows_behind(groups, 30), 6, 2, 48, 16, dtype, extra_stride=extra)
    run(ops, s, groups, 6, 2, 48, dtype)
    s.q = s.q[:, 1:] if extra > 1 else s.q           # and off 16 bytes
    run(ops, s, groups, 6, 2, 48, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sinks(ops, dtype):
    groups = [(3, 0), (4, 200), (1, 0)]
    positions = [0, 5, 40] + [199, 210, 260, 300] + [-1]
    s = make(groups, positions, 6, 3, 32, 16, dtype)
    run(ops, s, groups, 6, 3, 32, dtype, sink=1.5)
    run(ops, s, groups, 6, 3, 32, dtype, sink=torch.tensor([-3.0, 0.0, 1.0, 2.0, 30.0, -100.0], device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_see_nothing_give_zeros(ops, dtype):
    groups = [(3, 0), (2, 40)]
    s = make(groups, [-1, 3, -1, 40, 41], 4, 2, 64, 16, dtype)
    out, _ = run(ops, s, groups, 4, 2, 64, dtype, contexts=[0, 4, 70, 41, 42], most=42)
    assert (out[0] == 0).all() and (out[2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, n", [((8, 2, 64), 3), ((8, 2, 64), 24), ((16, 1, 48), 9), ((3, 3, 256), 5)])
@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("keys", [32, 1024])
def test_rows_that_see_nothing_beside_values_that_are_no_numbers(ops, keys, what, heads, n, dtype):
    """What is among the shared values reaches the rows that see it and not the padding between them."""
    Hq, Hkv, D = heads
    groups, positions = [(n, keys)], [keys + 7 * i for i in range(n)]
    s = make(groups, positions, *heads, 16, dtype)
    none = [1, n - 1]
    s.positions[none] = -1
    s.v[s.tables[0, 1], 0, 3, 5] = what                    # key 21, dim 3 of kv head 0
    step, group = step_of(s, most=max(positions) + 1)
    for share in (True, False, None):
        plan = ops[dtype].plan_shared_prefix(groups, [p + 1 for p in positions], *heads, share=share)
        for sink in (None, 0.5):
            got = ops[dtype].shared_prefix_attention(s.q, *heads, s.k, s.v, group, step, 0.1, plan, sink=sink).view(n, Hq, D).cpu()
            assert (got[none] == 0).all()
            got = got[[i for i in range(n) if i not in none]]
            reached = torch.zeros_like(got, dtype=torch.bool)
            reached[:, :Hq // Hkv, 3] = True
            assert torch.equal(~torch.isfinite(got), reached)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_plan_serves_later_steps(ops, dtype):
    """Contexts planned ahead: the positions of the step decide what is seen."""
    groups = [(6, 90), (2, 0)]
    for positions in ([90, 95, 100, 89, 110, 130, 0, 50], [189, 189, 189, 189, 189, 189, 189, 189], [89] * 6 + [31, 32]):
        s = make(groups, positions, 8, 2, 64, 16, dtype, seed=positions[0])
        s.tables = torch.cat([s.tables, torch.zeros((s.T, 8), dtype=torch.int32, device="cuda")], 1).contiguous()
        run(ops, s, groups, 8, 2, 64, dtype, contexts=[190] * 8)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-4, 1.0, 6.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_flat_and_sharp_weights(ops, dtype, scale):
    groups = [(9, 500)]
    s = make(groups, rows_behind(groups, 100), 4, 1, 64, 16, dtype)
    run(ops, s, groups, 4, 1, 64, dtype, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_growing_scores(ops, dtype):
    """Keys whose scores grow along the context: the running maximum moves on in every block."""
    groups = [(4, 400)]
    s = make(groups, [399, 420, 450, 500], 4, 2, 32, 16, dtype, poison=False)
    ramp = torch.zeros(s.k.shape[0], 16, device="cuda")
    for r in range(4):
        for j in range(int(s.positions[r]) + 1):
            ramp[s.tables[r, j // 16], j % 16] = j / 100.0
    s.k = (s.k.float() * 0.1 + ramp[:, None, :, None]).to(dtype)
    s.q = (s.q.float().abs()).to(dtype)
    run(ops, s, groups, 4, 2, 32, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_prefix_many_rows(ops, dtype):
    groups = [(70, 5000), (1, 0), (33, 2049)]
    s = make(groups, rows_behind(groups, 400, 3), 8, 2, 128, 16, dtype, poison=False)
    out, plan = run(ops, s, groups, 8, 2, 128, dtype)
    assert plan.column_tiles == (2 if dtype == BF16 else 1) and plan.join


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_as_paged_attention_and_the_same_bits_twice(ops, dtype):
    groups = [(12, 1000), (4, 0)]
    s = make(groups, rows_behind(groups, 200, 7), 8, 2, 64, 16, dtype)
    out, plan = run(ops, s, groups, 8, 2, 64, dtype)
    step, group = step_of(s)
    again = ops[dtype].shared_prefix_attention(s.q, 8, 2, 64, s.k, s.v, group, step, 0.125, plan)
    assert torch.equal(out, again)
    other = ops[dtype].paged_attention(s.q, 8, 2, 64, s.k, s.v, group, step, 0.125, None)
    check(other, *plain(s, 8, 2, 64, 0.125), 64, dtype)


@pytest.mark.gpu
def test_in_a_graph_and_on_another_stream(ops):
    groups = [(12, 700), (4, 0)]
    s = make(groups, [720 + i for i in range(12)] + [5, 90, 300, 719], 8, 2, 64, 16, BF16, poison=False)
    step, group = step_of(s, host={})
    plan = ops[BF16].plan_shared_prefix(groups, [p + 1 for p in s.positions.tolist()], 8, 2, 64, share=True)
    call = lambda: ops[BF16].shared_prefix_attention(s.q, 8, 2, 64, s.k, s.v, group, step, 0.125, plan)     # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = call()
    torch.cuda.synchronize()
    assert torch.equal(there, call())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        s.q.copy_(torch.randn(s.q.shape, generator=torch.Generator().manual_seed(i)))
        s.positions[12:].copy_(torch.tensor([5 - i, 90 - i, 300 - i, 719 - i]))
        s.positions[:12].sub_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        check(out, *plain(s, 8, 2, 64, 0.125), 64, BF16)


@pytest.mark.gpu
def test_a_plan_on_other_streams_and_not_in_a_capture(ops):
    """A plan made on one stream and used at once on another, thrown away while that still runs; none is made while a stream records."""
    groups = [(12, 700), (4, 0)]
    s = make(groups, [720 + i for i in range(12)] + [5, 90, 300, 719], 8, 2, 64, 16, BF16, poison=False)
    step, group = step_of(s)
    want = plain(s, 8, 2, 64, 0.125)
    contexts = [p + 1 for p in s.positions.tolist()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            plan = ops[BF16].plan_shared_prefix(groups, contexts, 8, 2, 64, share=True)
        with torch.cuda.stream(streams[1 - i % 2]):
            outs.append(ops[BF16].shared_prefix_attention(s.q, 8, 2, 64, s.k, s.v, group, step, 0.125, plan))
        del plan
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, outs[0])
    check(outs[0], *want, 64, BF16)
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="before a capture"):
            ops[BF16].plan_shared_prefix(groups, contexts, 8, 2, 64, share=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 2, 48)])
def test_table_entries_that_are_no_page(ops, heads, dtype):
    """Beyond a row's own pages a block table may hold anything."""
    groups = [(5, 96), (2, 0)]
    s = make(groups, [96, 100, 130, 140, 97, 3, 40], *heads, 16, dtype)
    s.tables = torch.cat([s.tables, torch.zeros((s.T, 9), dtype=torch.int32, device="cuda")], 1).contiguous()
    for r, p in enumerate(s.positions.tolist()):
        s.tables[r, p // 16 + 1:] = torch.tensor([-1, 2**31 - 1, -2**31, s.k.shape[0]], dtype=torch.int32).repeat(9)[:s.tables.shape[1] - p // 16 - 1].cuda()
    run(ops, s, groups, *heads, dtype)
    run(ops, s, groups, *heads, dtype, contexts=[200] * 7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (20, 1, 48), (4, 2, 256)])
@pytest.mark.parametrize("sink", [None, 0.5, "heads"])
def test_both_ways_into_the_kernels(ops, sink, heads, dtype):
    """The call that takes the tensors themselves and the one of plain numbers: the same results, the same refusals, nothing kept."""
    o = ops[dtype]
    groups = [(6, 100), (3, 0), (30, 48)]
    s = make(groups, rows_behind(groups, 60, 2), *heads, 16, dtype, extra_stride=8)
    step, group = step_of(s)
    contexts = [p + 1 for p in s.positions.tolist()]
    sink = torch.linspace(-1, 1, heads[0], device="cuda") if sink == "heads" else sink
    plans = [o.plan_shared_prefix(groups, contexts, *heads, share=share) for share in (True, False)]

    def call(**kw):
        a = {**dict(q=s.q, k=s.k, v=s.v, group=group, step=step, scale=0.2, plan=plans[0], sink=sink), **kw}
        return o.shared_prefix_attention(a["q"], *heads, a["k"], a["v"], a["group"], a["step"], a["scale"], a["plan"], sink=a["sink"])

    def refusals():
        for bad in (dict(q=s.q.double()), dict(q=s.q[:, :heads[0] * heads[2] - 1]), dict(q=s.q.t()), dict(k=s.k[:, :, :8]), dict(v=s.v.transpose(2, 3)),
                    dict(k=s.k.cpu()), dict(plan=SharedPrefixPlan(groups, contexts, *heads, "cpu", float32=dtype == F32)), dict(plan=None), dict(scale=math.inf),
                    dict(scale=0.0), dict(group=SimpleNamespace(block_tables=s.tables[:5])), dict(group=SimpleNamespace(block_tables=s.tables[:, :-1])),
                    dict(step=step_of(s, num_rows=4)[0]), dict(step=step_of(s, token_row=step.token_row[:-1])[0]), dict(step=step_of(s, most=10 ** 6)[0]),
                    dict(step=step_of(s, positions=step.positions.long())[0]), dict(sink=torch.zeros(heads[0] + 1, device="cuda"))):
            with pytest.raises((ValueError, TypeError)):
                call(**bad)

    call()
    short = [call(plan=p) for p in plans]
    held = [s.q, s.k, s.v, s.tables, step.positions, step.token_row, plans[0], plans[1]._data]
    before, memory = [sys.getrefcount(x) for x in held], torch.cuda.memory_allocated()
    for _ in range(20):
        call()
    refusals()
    assert [sys.getrefcount(x) for x in held] == before and torch.cuda.memory_allocated() == memory
    direct, o._direct = o._direct, SimpleNamespace(mie_direct_shared=lambda *args: None)
    try:
        refusals()
        for a, p in zip(short, plans):
            b = call(plan=p)
            assert a.dtype == b.dtype and torch.equal(a, b)
    finally:
        o._direct = direct


@pytest.mark.gpu
def test_a_step_of_no_rows(ops):
    plan = ops[BF16].plan_shared_prefix([], [], 4, 2, 64)
    assert (plan.num_items, plan.num_parts, plan.join) == (0, 0, False)
    s = make([(1, 0)], [4], 4, 2, 64, 16, BF16)
    step, group = step_of(s, most=0, num_rows=0, num_decode_rows=0, num_tokens=0, host={})
    step.token_row, step.positions = step.token_row[:0], step.positions[:0]
    assert ops[BF16].shared_prefix_attention(s.q[:0], 4, 2, 64, s.k, s.v, group, step, 0.1, plan).shape == (0, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_beyond_32_bits_of_offset(ops, dtype):
    Hq, Hkv, D, page = 4, 2, 128, 16
    pages = 2**31 // (Hkv * page * D) + 40                  # elements beyond 2^31
    k = torch.empty((pages, Hkv, page, D), dtype=dtype, device="cuda")
    v = torch.empty((pages, Hkv, D, page), dtype=dtype, device="cuda")
    small = make([(3, 40)], [45, 50, 39], Hq, Hkv, D, page, dtype, poison=False)
    far = small.tables + (pages - small.k.shape[0])
    k[pages - small.k.shape[0]:] = small.k
    v[pages - small.k.shape[0]:] = small.v
    step, _ = step_of(small)
    for share in (True, False):
        plan = ops[dtype].plan_shared_prefix([(3, 40)], [46, 51, 40], Hq, Hkv, D, share=share)
        out = ops[dtype].shared_prefix_attention(small.q, Hq, Hkv, D, k, v, SimpleNamespace(block_tables=far.contiguous()), step, 0.1, plan)
        check(out, *plain(small, Hq, Hkv, D, 0.1), D, dtype)


# ---- the plan, on the CPU

def covered(plan, groups, contexts, G):
    """Every key of every column exactly once, by the items; parts numbered in order."""
    items = plan.items.view(-1, 8).tolist()
    starts = plan.row_parts.tolist()
    seen = [[] for _ in range(len(contexts) * G)]
    wide = 64 * plan.column_tiles
    for row, columns, col0, begin, end, part, _, _ in items:
        assert begin < end and col0 % wide == 0 and col0 < columns and columns % G == 0
        for c in range(col0, min(columns, col0 + wide)):
            seen[row * G + c].append((begin, end, part))
    first = 0
    for n, keys in groups:
        for r in range(first, first + n):
            for h in range(G):
                parts = sorted(seen[r * G + h])
                assert [p for _, _, p in parts] == list(range(len(parts))) and len(parts) == starts[r + 1] - starts[r]
                at = 0
                for b, e, _ in parts:
                    assert b == at
                    at = e
                assert at == contexts[r]
        first += n
    assert plan.num_parts == starts[-1] and plan.join == any(b - a != 1 for a, b in zip(starts, starts[1:]))
    waves = items[plan.whole_items:]         # one row each, the longest first
    assert all(columns == G <= 16 for _, columns, *_ in waves) and [e - b for _, _, _, b, e, *_ in waves] == sorted((e - b for _, _, _, b, e, *_ in waves), reverse=True)
    first = 0
    for n, keys in groups:                   # an item of several rows holds shared keys only
        for row, columns, _, begin, end, _, _, _ in items:
            if row == first and columns > G:
                assert columns == n * G and end <= keys
        first += n


@pytest.mark.parametrize("share", [True, False, None])
@pytest.mark.parametrize("seed", range(40))
def test_a_plan_covers_every_key_once(seed, share):
    g = np.random.RandomState(seed)
    groups = [(int(g.randint(1, 40)), int(g.choice([0, 1, 31, 32, 500, 7000, 40000]))) for _ in range(g.randint(1, 6))]
    contexts = [k + int(g.choice([0, 1, 2, 33, 900])) for n, k in groups for _ in range(n)]
    G, Hkv = int(g.choice([1, 3, 8, 16])), int(g.choice([1, 4, 8]))
    plan = SharedPrefixPlan(groups, contexts, G * Hkv, Hkv, 64, "cpu", units=256 if seed < 30 else 4, float32=bool(seed % 2), share=share)
    covered(plan, groups, contexts, G)
    shared = any(columns > G for _, columns, *_ in plan.items.view(-1, 8).tolist())
    if share is not None:
        assert shared == (share and any(n > 1 and k > 0 for n, k in groups))


def test_a_plan_is_not_copied():
    plan = SharedPrefixPlan([(2, 5)], [6, 7], 4, 2, 64, "cpu")
    assert copy.deepcopy(plan) is plan
    with pytest.raises(TypeError, match="plan"):
        pickle.dumps(plan)
    with pytest.raises(TypeError, match="plan"):
        copy.copy(plan)


@pytest.mark.parametrize("bad", [([(2, 5)], [5, 4], 4, 2), ([(2, 5)], [5], 4, 2), ([(0, 5), (1, 0)], [5], 4, 2), ([(1, -1)], [5], 4, 2),
                                 ([(1, 0)], [-1], 4, 2), ([(1, 0)], [2**31], 4, 2), ([(1, 0)], [3], 5, 2), ([(1, 0)], [3], 5, 0)])
def test_refused_plans(bad):
    with pytest.raises(ValueError, match="shared prefix"):
        SharedPrefixPlan(*bad, 64, "cpu")


def test_refused_calls():
    """The checks come before anything is launched, so they are tried without a GPU."""
    b = object.__new__(HipBackend)
    groups, Hq, Hkv, D = [(3, 20)], 4, 2, 32
    s = make(groups, [20, 25, 30], Hq, Hkv, D, 16, BF16, device="cpu")
    step, group = step_of(s)
    plan = SharedPrefixPlan(groups, [21, 26, 31], Hq, Hkv, D, "cpu")
    ok = dict(qkv=s.q, Hq=Hq, Hkv=Hkv, D=D, k_cache=s.k, v_cache=s.v, group=group, step=step, scale=0.1, plan=plan)
    b._check_shared(**ok)

    def refused(error=ValueError, **kw):
        with pytest.raises(error):
            b._check_shared(**{**ok, **kw})

    refused(scale=0.0)
    refused(scale=-1.0)
    refused(scale=math.nan)
    refused(plan=None)
    refused(plan=SharedPrefixPlan([(2, 20)], [21, 26], Hq, Hkv, D, "cpu"))
    refused(plan=SharedPrefixPlan(groups, [21, 26, 31], Hq, 1, D, "cpu"))
    refused(plan=SharedPrefixPlan(groups, [21, 26, 3000], Hq, Hkv, D, "cpu"))     # beyond the block tables
    refused(plan=SharedPrefixPlan(groups, [21, 26, 30], Hq, Hkv, D, "cpu"))       # a row is further than planned
    refused(plan=SharedPrefixPlan(groups, [20, 31, 31], Hq, Hkv, D, "cpu"))
    refused(step=step_of(s, num_decode_rows=2)[0])
    refused(k_cache=s.k.float())
    refused(k_cache=s.k[:, :, :8])
    refused(qkv=s.q[:, :100])
    refused(qkv=s.q[:2])
    refused(group=SimpleNamespace(block_tables=s.tables.long()))
    pool = torch.zeros(s.k.numel() + 4, dtype=BF16)
    refused(k_cache=pool[4:].view(s.k.shape))
