"""The cases by which the serving operators are timed and checked: rotation of queries and keys, attention over
packed sequences, attention of requests that share a prefix.

`own` false: the plain forms, elementary torch operations in 32 bits (64 for angles), rounded once at the end.
`own` true: the calls that a user makes of this package.
"""

import math

import torch

own = False

HEAD_DIM = 128  # the head size that every attention entry point of this package takes


def _ints(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------------------------------------- cases
def _rotate(name, batch, tokens, heads, heads_kv, sections, interleaved, norm, fused, far):
    return {"name": name, "op": "rotate", "batch": batch, "tokens": tokens, "heads": heads, "heads_kv": heads_kv,
            "sections": sections, "interleaved": interleaved, "norm": norm, "fused": fused, "far": far}


def _packed(name, lens_q, lens_kv, heads, heads_kv, causal, lse, room):
    return {"name": name, "op": "packed", "lens_q": lens_q, "lens_kv": lens_kv, "heads": heads,
            "heads_kv": heads_kv, "causal": causal, "lse": lse, "room": room}


def _shared(name, prefix, lens_q, lens_kv, heads, heads_kv, lse, room):
    return {"name": name, "op": "shared", "prefix": prefix, "lens_q": lens_q, "lens_kv": lens_kv, "heads": heads,
            "heads_kv": heads_kv, "causal": True, "lse": lse, "room": room}


def _spread(count, low, high, step):
    """`count` lengths spread over low..high in a fixed order that is neither rising nor falling."""
    return ",".join(str(low + (i * step) % (high - low + 1)) for i in range(count))


def listed():
    return [
        # one decode step of 32 requests: new tokens at far positions of long texts
        _rotate("rotate_tokens", 1, 32, 32, 8, "64", False, True, False, 1000000),
        # a whole prompt batch of a text model with grouped heads
        _rotate("rotate_prompt", 1, 16384, 32, 8, "64", False, True, False, 0),
        # the video model's self-attention tokens: time, height and width positions, two samples
        _rotate("rotate_video", 2, 32768, 12, 12, "16,24,24", True, True, False, 0),
        # rows cut out of a fused q-k-v projection, no norm, a quarter of the pairs left unrotated, odd count
        _rotate("rotate_fused_rows", 1, 1537, 20, 4, "24,24", False, False, True, 5000),
        # a handful of short prompts: the smallest call, one of them with fewer keys than queries
        _packed("packed_short", "17,1,64,129,5", "17,1,64,129,3", 8, 2, True, True, False),
        # a prefill batch of prompts of very different lengths
        _packed("packed_prompts", "4096,2311,1,777,8192,129,530,1500", "4096,2311,1,777,8192,129,530,1500",
                32, 8, True, False, False),
        # later chunks of long prompts: queries in the middle of a text, history in the cache
        _packed("packed_chunks", "512,512,333,512", "4608,9728,2381,16896", 32, 4, True, False, True),
        # video clips of different lengths in one batch, every token sees its whole clip
        _packed("packed_clips", "9000,4097,12288", "9000,4097,12288", 12, 12, False, False, False),
        # the longest single prompt, without grouping, with the log-sum-exp
        _packed("packed_long", "16384", "16384", 16, 16, True, True, False),
        # a decode step: one token per request against its own cache
        _packed("packed_tokens", ",".join(["1"] * 64), _spread(64, 100, 12000, 4463), 32, 8, True, False, True),
        # few requests behind a short system prompt: latency
        _shared("shared_few", 1000, "1,1,1,1", "1,37,64,12", 16, 4, True, True),
        # a serving batch behind one long document
        _shared("shared_document", 32768, ",".join(["1"] * 64), _spread(64, 1, 1024, 389), 32, 8, False, True),
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def _draw_once(rng):
    op = rng.choice(["rotate", "packed", "packed", "shared"])
    heads_kv = rng.choice([1, 2, 4, 6, 8, 12])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    heads = heads_kv * group
    if op == "rotate":
        cuts = rng.choice(["64", "16,24,24", "24,24", "20,22,22", "32", "10,21,30"])
        batch = rng.choice([1, 1, 2, 3])
        return _rotate("", batch, _log_int(rng, 1, 32768 // batch), heads, heads_kv, cuts, rng.random() < 0.5,
                       rng.random() < 0.7, rng.random() < 0.4, rng.choice([0, 5000, 1000000]))
    if op == "shared":
        count = _log_int(rng, 1, 96)
        lens_q = [rng.choice([1, 1, 1, 1, 2, 4]) for _ in range(count)]
        longest = _log_int(rng, 4, 1500)
        lens_kv = [n + rng.randint(0, longest) for n in lens_q]
        return _shared("", _log_int(rng, 1, 32768), ",".join(map(str, lens_q)), ",".join(map(str, lens_kv)), heads,
                       heads_kv, rng.random() < 0.5, rng.random() < 0.5)
    kind = rng.choice(["prompts", "prompts", "chunks", "tokens", "clips"])
    if kind == "tokens":
        count = _log_int(rng, 1, 96)
        longest = _log_int(rng, 1, 16384)
        lens_q, lens_kv = [1] * count, [rng.randint(1, longest) for _ in range(count)]
    else:
        count = _log_int(rng, 1, 24)
        longest = _log_int(rng, 2, 12000)
        lens_q = [_log_int(rng, 1, longest) for _ in range(count)]
        lens_kv = [n + (_log_int(rng, 1, 12000) if kind == "chunks" else 0) for n in lens_q]
    return _packed("", ",".join(map(str, lens_q)), ",".join(map(str, lens_kv)), heads, heads_kv, kind != "clips",
                   rng.random() < 0.5, kind in ("tokens", "chunks"))


def draw(rng):
    top = {}
    for case in listed():
        w = work(case)
        old = top.get(case["op"], (0, 0))
        top[case["op"]] = (max(old[0], w["bytes"]), max(old[1], w["flops"]))
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] <= top[case["op"]][0] and w["flops"] <= top[case["op"]][1]:
            return case


# ------------------------------------------------------------------------------------------------- work
def _pairs(lens_q, lens_kv, causal):
    """(query, key) pairs that see each other."""
    total = 0
    for n, m in zip(lens_q, lens_kv):
        if causal:
            first = max(0, n - m)  # queries before this one see nothing
            total += sum(range(m - n + first + 1, m + 1))
        else:
            total += n * m
    return total


def work(case):
    h, hk = case["heads"], case["heads_kv"]
    row = HEAD_DIM * 2
    if case["op"] == "rotate":
        t = case["batch"] * case["tokens"]
        values = t * (h + hk) * HEAD_DIM
        axes = len(_ints(case["sections"]))
        # a square and a sum, two products of the norm, three operations of the rotation for each value
        return {"bytes": 2 * values * 2 + t * axes * 8, "flops": values * (7 if case["norm"] else 3)}
    lq, lk = _ints(case["lens_q"]), _ints(case["lens_kv"])
    tokens = sum(lq)
    rows_kv = sum(lk) + case.get("prefix", 0)
    pairs = _pairs(lq, lk, case["causal"]) + tokens * case.get("prefix", 0)
    size = 2 * tokens * h * row + 2 * rows_kv * hk * row + (tokens * h * 4 if case["lse"] else 0)
    return {"bytes": size, "flops": 4 * HEAD_DIM * h * pairs}


# ------------------------------------------------------------------------------------------------- inputs
def _starts(lens, room):
    """First row of each sequence in the K/V rows: back to back, or with room to grow up to the next multiple of 256."""
    starts, at = [], 0
    for n in lens:
        starts.append(at)
        at += (n // 256 + 1) * 256 if room else n
    return starts, max(at, 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    h, hk = case["heads"], case["heads_kv"]

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    state = {"case": case}
    if case["op"] == "rotate":
        b, t = case["batch"], case["tokens"]
        if case["fused"]:  # q, k and v of a token lie side by side
            rows = rand(b, t, h + 2 * hk, HEAD_DIM)
            state["q"], state["k"] = rows[:, :, :h], rows[:, :, h:h + hk]
        else:
            state["q"], state["k"] = rand(b, t, h, HEAD_DIM), rand(b, t, hk, HEAD_DIM)
        sections = _ints(case["sections"])
        if len(sections) == 3:  # a video: width fastest
            width = max(1, math.isqrt(t // 8)) if t >= 8 else 1
            i = torch.arange(t, device="cuda")
            pos = torch.stack([i // (width * width), i // width % width, i % width])
        else:
            pos = torch.arange(t, device="cuda").repeat(len(sections), 1)
        shift = torch.randint(0, case["far"] + 1, (len(sections), 1), generator=gen, device="cuda")
        state["positions"] = (pos + shift).contiguous()
        # each axis has a falling series of frequencies of its own
        state["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float32) / n)
                                       for n in sections])
        state["sections"] = tuple(sections)
        if case["norm"]:
            state["q_weight"] = (1 + 0.2 * torch.randn(HEAD_DIM, generator=gen, device="cuda")).to(torch.bfloat16)
            state["k_weight"] = (1 + 0.2 * torch.randn(HEAD_DIM, generator=gen, device="cuda")).to(torch.bfloat16)
        else:
            state["q_weight"] = state["k_weight"] = None
        return state
    lq, lk = _ints(case["lens_q"]), _ints(case["lens_kv"])
    starts, rows = _starts(lk, case["room"])
    state.update(lens_q=lq, lens_kv=lk, starts=starts, q=rand(sum(lq), h, HEAD_DIM), k=rand(rows, hk, HEAD_DIM),
                 v=rand(rows, hk, HEAD_DIM))
    if case["op"] == "shared":
        state.update(k_prefix=rand(case["prefix"], hk, HEAD_DIM), v_prefix=rand(case["prefix"], hk, HEAD_DIM))
    if own:
        from b200_attention_b200 import ops

        state["plan"] = ops.AttentionPlan(lq, lk, heads=h, heads_kv=hk, causal=case["causal"], starts_kv=starts,
                                          len_prefix=case.get("prefix", 0), device="cuda")
    return state


# ------------------------------------------------------------------------------------------------- plain forms
EPS = 1e-6


def _plain_rotate(s):
    case = s["case"]
    axis = [a for a, n in enumerate(s["sections"]) for _ in range(n)]
    angle = s["positions"].double()[axis].T * s["inv_freq"].double()  # [T, pairs]
    pad = HEAD_DIM // 2 - angle.shape[1]
    cos = torch.nn.functional.pad(torch.cos(angle), (0, pad), value=1.0).float()[None, :, None]
    sin = torch.nn.functional.pad(torch.sin(angle), (0, pad), value=0.0).float()[None, :, None]
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        if case["interleaved"]:
            a, b = x[..., 0::2], x[..., 1::2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :HEAD_DIM // 2], x[..., HEAD_DIM // 2:]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(y.to(torch.bfloat16))
    return out


def _plain_rows(q, k, v, visible):
    """q [H, n, 128], k and v [Hkv, m, 128] in 32 bits; visible [n, m] or None. A block of query rows at a time."""
    h, n, _ = q.shape
    hk, m, _ = k.shape
    group = h // hk
    q = q.reshape(hk, group, n, HEAD_DIM)
    step = max(1, (1 << 28) // max(1, h * m))
    outs, lses = [], []
    for i in range(0, n, step):
        s = torch.matmul(q[:, :, i:i + step].reshape(hk, -1, HEAD_DIM), k.transpose(1, 2)) / math.sqrt(HEAD_DIM)
        s = s.reshape(hk, group, -1, m)
        if visible is not None:
            s = s.masked_fill(~visible[i:i + step], -math.inf)
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.reshape(hk, -1, m), v).reshape(hk, group, -1, HEAD_DIM)
        o = torch.where(total > 0, o / total, torch.zeros_like(o))
        outs.append(o.reshape(h, -1, HEAD_DIM))
        lses.append((top + torch.log(total)).reshape(h, -1))
    return torch.cat(outs, 1), torch.cat(lses, 1)


def _plain_attention(s):
    case = s["case"]
    prefix = case.get("prefix", 0)
    o = torch.empty_like(s["q"])
    lse = torch.empty(case["heads"], s["q"].shape[0], device="cuda")
    at = 0
    for n, m, start in zip(s["lens_q"], s["lens_kv"], s["starts"]):
        k, v = s["k"][start:start + m], s["v"][start:start + m]
        if case["op"] == "shared":
            k, v = torch.cat([s["k_prefix"], k]), torch.cat([s["v_prefix"], v])
        total = m + prefix
        visible = None
        if case["causal"]:
            i = torch.arange(n, device="cuda")[:, None]
            visible = torch.arange(total, device="cuda")[None] <= i + (total - n)
        oi, li = _plain_rows(s["q"][at:at + n].float().transpose(0, 1), k.float().transpose(0, 1),
                             v.float().transpose(0, 1), visible)
        o[at:at + n] = oi.transpose(0, 1).to(torch.bfloat16)
        lse[:, at:at + n] = li
        at += n
    return [o, lse] if case["lse"] else o


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return _plain_rotate(state) if case["op"] == "rotate" else _plain_attention(state)
    from b200_attention_b200 import ops

    if case["op"] == "rotate":
        return ops.qk_norm_rope(state["q"], state["k"], state["positions"], state["inv_freq"],
                                sections=state["sections"], q_weight=state["q_weight"], k_weight=state["k_weight"],
                                eps=EPS, interleaved=case["interleaved"])
    if case["op"] == "packed":
        return ops.attention_packed(state["q"], state["k"], state["v"], state["plan"], return_lse=case["lse"])
    return ops.attention_shared_prefix(state["q"], state["k_prefix"], state["v_prefix"], state["k"], state["v"],
                                       state["plan"], return_lse=case["lse"])


# ------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """What `run` returns, from the definitions, in 64 bits: one head, or one request, at a time."""
    s = prepare(case, seed)
    if case["op"] == "rotate":
        result = []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / HEAD_DIM + EPS) * w.double()
            y = x.clone()
            j = 0
            for axis, n in enumerate(s["sections"]):
                for _ in range(n):
                    a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + HEAD_DIM // 2)
                    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                                       s["positions"][axis].double() * s["inv_freq"][j].double())
                    z = torch.complex(x[..., a], x[..., b]) * turn[None, :, None]
                    y[..., a], y[..., b] = z.real, z.imag
                    j += 1
            result.append(y)
        return result
    if work(case)["flops"] > 4e12:
        return None
    group = case["heads"] // case["heads_kv"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((case["heads"], s["q"].shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    prefix = case.get("prefix", 0)
    at = 0
    for n, m, start in zip(s["lens_q"], s["lens_kv"], s["starts"]):
        total = prefix + m
        for g in range(case["heads_kv"]):
            k, v = s["k"][start:start + m, g].double(), s["v"][start:start + m, g].double()
            if prefix:
                k, v = torch.cat([s["k_prefix"][:, g].double(), k]), torch.cat([s["v_prefix"][:, g].double(), v])
            if total == 0:
                continue
            step = max(1, (1 << 27) // (group * total))
            for i in range(0, n, step):
                e = min(n, i + step)
                qi = s["q"][at + i:at + e, g * group:(g + 1) * group].double()  # [rows, group, 128]
                logits = torch.einsum("rgd,md->grm", qi, k) * HEAD_DIM ** -0.5
                if case["causal"]:
                    last = torch.arange(i, e, device="cuda") + total - n  # last key that each row sees
                    logits.masked_fill_(torch.arange(total, device="cuda") > last[:, None], -math.inf)
                li = torch.logsumexp(logits, -1)  # [group, rows]
                weight = torch.exp(logits - torch.where(li == -math.inf, 0.0, li)[..., None])
                o[at + i:at + e, g * group:(g + 1) * group] = torch.einsum("grm,md->rgd", weight, v)
                lse[g * group:(g + 1) * group, at + i:at + e] = li
        at += n
    return [o, lse] if case["lse"] else o
