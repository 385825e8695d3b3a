"""Operators of a step that answers one prompt many times: attention of single tokens whose requests share the first part
of their cache, and the choice of the next tokens under each request's own rules (penalties for tokens already there,
biases on single tokens, masks of what a grammar allows).

``own`` False: the operators in elementary torch operations.  ``own`` True: the calls a user makes of the framework.
"""
import math

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # four answers to a short prompt, a few tokens in: nothing but launches
        dict(name="shared, 4 rows of 200 keys", op="shared", dtype="bf16", q_heads=32, kv_heads=4, dim=64, groups=1, rows=4, prefix=200, own_keys=40),
        # thirty-two answers to a prompt of one page of text
        dict(name="shared, 32 rows of 2000 keys", op="shared", dtype="bf16", q_heads=32, kv_heads=8, dim=128, groups=1, rows=32, prefix=2000, own_keys=512),
        # a few answers to a long document
        dict(name="shared, 8 rows of 30000 keys", op="shared", dtype="bf16", q_heads=32, kv_heads=8, dim=128, groups=1, rows=8, prefix=30000, own_keys=700),
        # eight prompts of different lengths with eight answers each
        dict(name="shared, 8 times 8 rows", op="shared", dtype="bf16", q_heads=32, kv_heads=4, dim=64, groups=8, rows=8, prefix=3500, own_keys=900),
        # a full batch behind one system prompt with its documents
        dict(name="shared, 256 rows of 8192 keys", op="shared", dtype="bf16", q_heads=32, kv_heads=8, dim=128, groups=1, rows=256, prefix=8192, own_keys=1024),
        # the 32-bit engine: twenty-four answers
        dict(name="shared, float32, 24 rows", op="shared", dtype="f32", q_heads=32, kv_heads=4, dim=64, groups=1, rows=24, prefix=1500, own_keys=100),
        # one request's next token: nothing but launches
        dict(name="choose, 1 row of 32000", op="choose", rows=1, vocab=32000, history=300, masked=0, biased=20),
        # an ordinary batch, some of it under a grammar
        dict(name="choose, 32 rows of 32000", op="choose", rows=32, vocab=32000, history=2000, masked=12, biased=30),
        # a vocabulary that is no multiple of anything, everything under a grammar
        dict(name="choose, 7 rows of 50261", op="choose", rows=7, vocab=50261, history=5000, masked=7, biased=300),
        # a full batch of a large vocabulary
        dict(name="choose, 256 rows of 128256", op="choose", rows=256, vocab=128256, history=2000, masked=64, biased=50),
        # logits for a caller that chooses itself
        dict(name="adjust, 8 rows of 32000", op="adjust", rows=8, vocab=32000, history=1000, masked=4, biased=10),
        # and a full batch with long histories
        dict(name="adjust, 192 rows of 128256", op="adjust", rows=192, vocab=128256, history=12000, masked=96, biased=300),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        dim = rng.choice([16, 32, 64, 64, 96, 128, 128, 256])
        kv = rng.randint(1, 8)
        group = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
        dtype = "f32" if rng.random() < 0.25 else "bf16"
        groups = rng.choice([1, 1, 2, 3, 5, 8])
        rows = _spread(rng, 1, max(1, 256 // groups))
        own_keys = _spread(rng, 1, max(2, min(1024, (800 * 256 * 8 * 128) // (groups * rows * kv * dim * (2 if dtype == "f32" else 1)))))
        most = (8192 * 256 * 32 * 128) // (groups * rows * kv * group * dim * (4 if dtype == "f32" else 1))
        return dict(op="shared", dtype=dtype, q_heads=kv * group, kv_heads=kv, dim=dim, groups=groups, rows=rows,
                    prefix=_spread(rng, 1, max(2, min(32768 // groups, most))), own_keys=own_keys)
    rows = _spread(rng, 1, 192)
    return dict(op=rng.choice(["choose", "adjust"]), rows=rows, vocab=_spread(rng, 1000, 128256), history=_spread(rng, 1, 12000),
                masked=rng.randint(0, rows), biased=_spread(rng, 1, 300))


# ------------------------------------------------------------------ attention over a shared first part


def _lengths(case, seed):
    """Shared keys of every group and positions of every row, on the host."""
    g = torch.Generator().manual_seed(seed)
    G, n, P = case["groups"], case["rows"], case["prefix"]
    low = P if G == 1 else max(1, (3 * P) // 5)
    keys = torch.randint(low, P + 1, (G,), generator=g)
    mine = torch.randint(1, case["own_keys"] + 1, (G, n), generator=g)
    return keys, keys[:, None] + mine - 1


def _prepare_shared(case, seed):
    keys, pos = _lengths(case, seed)
    G, n, Hq, Hkv, D = case["groups"], case["rows"], case["q_heads"], case["kv_heads"], case["dim"]
    dt, dev = DTYPES[case["dtype"]], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    blocks = int(pos.max()) // PAGE + 1
    whole = keys // PAGE                                          # pages that lie wholly within the shared keys
    need = pos // PAGE + 1 - whole[:, None]                       # pages a row has of its own
    total = 1 + int(whole.sum()) + int(need.sum())
    ids = torch.randperm(total - 1, generator=torch.Generator().manual_seed(seed + 1)) + 1      # page 0 is scratch
    tables = torch.zeros((G, n, blocks), dtype=torch.int64)
    at = 0
    for i in range(G):
        w = int(whole[i])
        tables[i, :, :w] = ids[at:at + w]
        at += w
        for r in range(n):
            k = int(need[i, r])
            tables[i, r, w:w + k] = ids[at:at + k]
            at += k
    # keys with a common part, as rotated keys have, and values with a mean of their own a channel
    base = torch.randn((1, Hkv, 1, D), generator=g, device=dev)
    mean = torch.randn((1, Hkv, D, 1), generator=g, device=dev) * 0.5
    k_cache = torch.randn((total, Hkv, PAGE, D), generator=g, device=dev, dtype=dt).add_(base.to(dt))
    v_cache = torch.randn((total, Hkv, D, PAGE), generator=g, device=dev, dtype=dt).add_(mean.to(dt))
    dtab = tables.to(dev)
    for i in range(G):                                            # the page in which the shared keys end: a copy a row
        w, r = int(whole[i]), int(keys[i]) % PAGE
        if r:
            k_cache[dtab[i, 1:, w], :, :r] = k_cache[dtab[i, 0, w], :, :r].clone()
            v_cache[dtab[i, 1:, w], :, :, :r] = v_cache[dtab[i, 0, w], :, :, :r].clone()
    T = G * n
    state = dict(case=case, q=(1.5 * torch.randn((T, Hq * D), generator=g, device=dev)).to(dt), k_cache=k_cache, v_cache=v_cache,
                 tables=dtab.view(T, blocks).to(torch.int32), positions=pos.view(T).to(torch.int32).to(dev),
                 keys=keys.to(torch.int32).to(dev), scale=D ** -0.5, longest=int(keys.max()), host_keys=keys.tolist(),
                 host_positions=pos.view(T).tolist())
    if own:                         # what an engine keeps from step to step: the step's arrays and the plan of who shares what
        from mini_inference_engine_amd.engine.batch import GroupStep, StepContext
        ramp = torch.arange(T + 1, dtype=torch.int32, device=dev)
        most = int(pos.max()) + 1
        state["step"] = StepContext(
            num_tokens=T, num_rows=T, num_decode_rows=T, num_logits=T, input_ids=ramp[:T], positions=state["positions"], token_row=ramp[:T],
            row_start=ramp, row_position=state["positions"], row_context=state["positions"] + 1, state_slots=ramp[:T], logit_rows=ramp[:T],
            page_size=PAGE, max_row_tokens=1, max_context=most)
        state["group"] = GroupStep(state["tables"], ramp[:T], blocks)
        state["plan"] = _backend(dt).plan_shared_prefix([(n, k) for k in state["host_keys"]], [p + 1 for p in state["host_positions"]],
                                                        Hq, Hkv, D)
    return state


def _shared_plain(s):
    c, P = s["case"], PAGE
    G, n, Hq, Hkv, D = c["groups"], c["rows"], c["q_heads"], c["kv_heads"], c["dim"]
    h, T = Hq // Hkv, G * n
    tables, keys, dev = s["tables"].long(), s["keys"].long(), s["q"].device
    q = s["q"].float().view(G, n, Hkv, h, D) * s["scale"]
    # the shared keys, once a group
    first = tables.view(G, n, -1)[:, 0, :(s["longest"] + P - 1) // P]
    L = first.shape[1] * P
    k = s["k_cache"][first].float().permute(0, 2, 1, 3, 4).reshape(G, Hkv, L, D)
    v = s["v_cache"][first].float().permute(0, 2, 1, 4, 3).reshape(G, Hkv, L, D)
    z1 = q.permute(0, 2, 1, 3, 4).reshape(G, Hkv, n * h, D) @ k.transpose(2, 3)
    z1 = z1.masked_fill_((torch.arange(L, device=dev) >= keys[:, None])[:, None, None], -math.inf)
    z1 = z1.view(G, Hkv, n, h, L).transpose(1, 2).reshape(T, Hkv, h, L)
    # every row's own keys, from the page in which the shared ones end
    begin = (keys // P).repeat_interleave(n)
    blocks = c["own_keys"] // P + 2
    at = begin[:, None] + torch.arange(blocks, device=dev)
    mine = tables.gather(1, at.clamp(max=tables.shape[1] - 1))
    M = blocks * P
    k2 = s["k_cache"][mine].float().permute(0, 2, 1, 3, 4).reshape(T, Hkv, M, D)
    v2 = s["v_cache"][mine].float().permute(0, 2, 1, 4, 3).reshape(T, Hkv, M, D)
    place = begin[:, None] * P + torch.arange(M, device=dev)
    seen = (place >= keys.repeat_interleave(n)[:, None]) & (place <= s["positions"].long()[:, None])
    z2 = (q.view(T, Hkv, h, D) @ k2.transpose(2, 3)).masked_fill_(~seen[:, None, None], -math.inf)
    most = torch.maximum(z1.amax(-1, keepdim=True), z2.amax(-1, keepdim=True))
    w1, w2 = torch.exp(z1 - most), torch.exp(z2 - most)
    total = w1.sum(-1, keepdim=True) + w2.sum(-1, keepdim=True)
    o1 = w1.view(G, n, Hkv, h, L).transpose(1, 2).reshape(G, Hkv, n * h, L) @ v
    o1 = o1.view(G, Hkv, n, h, D).transpose(1, 2).reshape(T, Hkv, h, D)
    return ((o1 + w2 @ v2) / total).reshape(T, Hq * D).to(s["q"].dtype)


def _shared_exact(s):
    c, P = s["case"], PAGE
    n, Hq, Hkv, D = c["rows"], c["q_heads"], c["kv_heads"], c["dim"]
    out = []
    for row, p in enumerate(s["host_positions"]):
        pages = s["tables"][row, :p // P + 1].long()
        k = s["k_cache"][pages].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :p + 1]
        v = s["v_cache"][pages].double().permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :p + 1]
        q = s["q"][row].double().view(Hkv, Hq // Hkv, D)
        w = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D), dim=-1)
        out.append(torch.matmul(w, v).reshape(Hq * D))
    return torch.stack(out)


# ------------------------------------------------------------------ rules on logits


def _prepare_rules(case, seed):
    R, V, dev = case["rows"], case["vocab"], "cuda"
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=dev).manual_seed(seed)
    slots, most = R + 3, case["history"] + 5
    # texts repeat themselves: a token's rank falls off like one over it
    rank = torch.rand((slots, most), generator=gd, device=dev, dtype=torch.float64)
    history = torch.exp(rank * math.log(V)).long().sub_(1).clamp_(0, V - 1)
    history = (history * 7919 + 13) % V
    lengths = torch.randint(max(1, case["history"] // 3), case["history"] + 1, (R,), generator=g)
    prompt = (lengths * torch.rand(R, generator=g)).long()
    on = torch.rand(R, generator=g) < 0.75
    repetition = torch.where(on, 1.0 + 0.5 * torch.rand(R, generator=g), torch.ones(R))
    presence = torch.where(on, torch.rand(R, generator=g) * 1.5 - 0.25, torch.zeros(R))
    frequency = torch.where(on, torch.rand(R, generator=g) * 0.75, torch.zeros(R))
    # biases: some tokens a row, none twice
    count = torch.randint(0, case["biased"] + 1, (R,), generator=g)
    starts = torch.zeros(R + 1, dtype=torch.int64)
    starts[1:] = count.cumsum(0)
    N = int(starts[-1])
    step = torch.randint(1, max(2, V // (case["biased"] + 1)), (R,), generator=g)
    of = torch.repeat_interleave(torch.arange(R), count)
    tokens = (torch.arange(N) - starts[of]) * step[of]
    values = torch.randn(N, generator=g) * 4
    # masks: of the first ``masked`` rows; some let few tokens through, one nothing, the rest about half
    M, words = case["masked"], (V + 31) // 32
    masks = torch.randint(-2**31, 2**31, (max(1, M), words), generator=gd, device=dev, dtype=torch.int64)
    few = torch.arange(max(1, M), device=dev) % 3 == 1
    masks = torch.where(few[:, None] & (torch.arange(words, device=dev) % 97 != 5), torch.zeros_like(masks), masks)
    if M > 4:
        masks[4] = 0
    mask_rows = torch.full((R,), -1, dtype=torch.int64)
    mask_rows[torch.randperm(R, generator=g)[:M]] = torch.arange(M)
    logits = 3 * torch.randn((R, V), generator=gd, device=dev)
    if M:                           # what a mask hides may be anything
        hidden = (masks[0][torch.arange(V, device=dev) // 32] >> (torch.arange(V, device=dev) % 32)) & 1 == 0
        logits[int((mask_rows == 0).nonzero()[0, 0]), hidden] = math.nan
    i32, f32 = (lambda t: t.to(torch.int32).to(dev)), (lambda t: t.float().to(dev))
    temperatures = torch.where(torch.rand(R, generator=g) < 0.25, 0.5 + torch.rand(R, generator=g), torch.zeros(R))
    return dict(case=case, logits=logits, out=torch.empty_like(logits), history=i32(history), slots=i32(torch.randperm(slots - 1, generator=g)[:R] + 1),
                lengths=i32(lengths), prompt=i32(prompt), repetition=f32(repetition), presence=f32(presence), frequency=f32(frequency),
                bias_starts=i32(starts), bias_tokens=i32(tokens), bias_values=f32(values), masks=i32(masks), mask_rows=i32(mask_rows),
                temperatures=f32(temperatures), seeds=torch.randint(0, 2**62, (R,), generator=g).to(dev),
                counters=i32(lengths - prompt), bias_rows=i32(of), plan=None)


def _adjust_plain(s):
    z, R, V = s["logits"], s["logits"].shape[0], s["logits"].shape[1]
    rows = s["history"][s["slots"].long()]
    at = torch.arange(rows.shape[1], device=z.device)
    known = (at < s["lengths"][:, None]).float()
    output = known * (at >= s["prompt"][:, None]).float()
    ids = rows.long()
    there = torch.zeros((R, V), device=z.device).scatter_add_(1, ids, known) > 0
    times = torch.zeros((R, V), device=z.device).scatter_add_(1, ids, output)
    rep = s["repetition"][:, None]
    z = torch.where(there, torch.where(z > 0, z / rep, z * rep), z)
    z = z - s["frequency"][:, None] * times
    z = z - s["presence"][:, None] * (times > 0).float()
    bias = torch.zeros((R, V), device=z.device)
    bias[s["bias_rows"].long(), s["bias_tokens"].long()] = s["bias_values"]
    z = z + bias
    v = torch.arange(V, device=z.device)
    words = s["masks"][s["mask_rows"].clamp(min=0).long()]
    allowed = (words[:, v // 32] >> (v % 32)) & 1
    return torch.where((allowed > 0) | (s["mask_rows"][:, None] < 0), z, torch.full_like(z, -math.inf))


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _uniform(s, V):
    """The uniform numbers of (seed, counter, token), as sampling without rules draws them."""
    seed = s["seeds"]
    key = _mix(_mix(_mix(seed & 0xFFFFFFFF) ^ ((seed >> 32) & 0xFFFFFFFF)) ^ s["counters"].long())
    x = _mix(key[:, None] ^ _mix((torch.arange(V, device=seed.device) + 0x9E3779B9) & 0xFFFFFFFF))
    return ((x >> 9).double() + 0.5) * 2.0 ** -23


def _choose_plain(s):
    z = _adjust_plain(s)
    V = z.shape[1]
    t = s["temperatures"].double()[:, None]
    drawn = z.double() / torch.where(t > 0, t, torch.ones_like(t)) - torch.log(-torch.log(_uniform(s, V)))      # 64 bits: next to a border
    z = torch.where(t > 0, drawn, z.double())
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    best = z.amax(1, keepdim=True)
    return torch.where(z == best, torch.arange(V, device=z.device), V).amin(1).to(torch.int32)


def _adjust_exact(s):
    out = []
    for r in range(s["logits"].shape[0]):
        z = s["logits"][r].double()
        V = z.shape[0]
        text = s["history"][int(s["slots"][r]), :int(s["lengths"][r])].long()
        p = float(s["repetition"][r])
        seen = torch.unique(text)
        z[seen] = torch.where(z[seen] > 0, z[seen] / p, z[seen] * p)
        new, times = torch.unique(text[int(s["prompt"][r]):], return_counts=True)
        z[new] -= float(s["frequency"][r]) * times.double() + float(s["presence"][r])
        a, b = int(s["bias_starts"][r]), int(s["bias_starts"][r + 1])
        z[s["bias_tokens"][a:b].long()] += s["bias_values"][a:b].double()
        m = int(s["mask_rows"][r])
        if m >= 0:
            bits = (s["masks"][m].long()[:, None] >> torch.arange(32, device=z.device)) & 1
            z[bits.reshape(-1)[:V] == 0] = -math.inf
        out.append(z)
    return out


def _choose_exact(s):
    chosen = []
    noise = -torch.log(-torch.log(_uniform(s, s["logits"].shape[1])))
    for r, z in enumerate(_adjust_exact(s)):
        t = float(s["temperatures"][r])
        z = torch.nan_to_num(z if t == 0 else z / t + noise[r], nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        chosen.append(int((z == z.max()).nonzero()[0, 0]))
    return torch.tensor(chosen, dtype=torch.int32)


# ------------------------------------------------------------------ the framework's calls

_backends = {}


def _backend(dtype):
    if dtype not in _backends:
        from mini_inference_engine_amd.kernels.hip_backend import HipBackend
        _backends[dtype] = HipBackend(dtype)
    return _backends[dtype]


def _rules(s):
    from mini_inference_engine_amd.kernels.api import LogitRules
    return LogitRules(history=s["history"], slots=s["slots"], lengths=s["lengths"], prompt_lengths=s["prompt"], repetition=s["repetition"],
                      presence=s["presence"], frequency=s["frequency"], bias_starts=s["bias_starts"], bias_tokens=s["bias_tokens"],
                      bias_values=s["bias_values"], masks=s["masks"], mask_rows=s["mask_rows"])


def prepare(case, seed):
    return _prepare_shared(case, seed) if case["op"] == "shared" else _prepare_rules(case, seed)


def run(state):
    c = state["case"]
    if c["op"] == "shared":
        if own:
            return _backend(DTYPES[c["dtype"]]).shared_prefix_attention(
                state["q"], c["q_heads"], c["kv_heads"], c["dim"], state["k_cache"], state["v_cache"], state["group"], state["step"],
                state["scale"], state["plan"])
        return _shared_plain(state)
    if c["op"] == "adjust":
        return _backend(torch.bfloat16).adjust_logits(state["logits"], _rules(state), out=state["out"]) if own else _adjust_plain(state)
    if own:
        return _backend(torch.bfloat16).sample(state["logits"], state["temperatures"], state["seeds"], state["counters"], rules=_rules(state))
    return _choose_plain(state)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "shared":
        return _shared_exact(s)
    return torch.stack(_adjust_exact(s)) if case["op"] == "adjust" else _choose_exact(s)


def work(case):
    if case["op"] == "shared":
        # sizes are drawn: the mean of what they are drawn from
        size = 4 if case["dtype"] == "f32" else 2
        T = case["groups"] * case["rows"]
        prefix = case["prefix"] * (1.0 if case["groups"] == 1 else 0.8)
        mine = (case["own_keys"] + 1) / 2
        kv = (case["groups"] * prefix + T * mine) * 2 * case["kv_heads"] * case["dim"] * size
        return {"bytes": int(kv + 2 * T * case["q_heads"] * case["dim"] * size),
                "flops": int(4 * T * (prefix + mine) * case["q_heads"] * case["dim"])}
    R, V = case["rows"], case["vocab"]
    read = R * V * 4 + case["masked"] * V / 8 + R * case["history"] * 4 * 2 / 3 + R * case["biased"] * 4
    if case["op"] == "adjust":
        return {"bytes": int(read + R * V * 4), "flops": 4 * R * V}
    return {"bytes": int(read + R * 4), "flops": 6 * R * V}
