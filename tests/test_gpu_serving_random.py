"""GPU tests: packed, shared-prefix and rotation calls of random shapes against the plain 64-bit forms.

A few cases of fixed seeds here; `python -m tests.test_gpu_serving_random COUNT [SEED]` runs COUNT of each kind."""

import math
import random
import sys

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu


def rand(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def draw_attention(rng):
    """Head counts, lengths, order in the cache, mask, prefix, rows that are nobody's; of limited cost."""
    while True:
        heads_kv, group = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 11, 16, 33, 64, 128])
        heads = heads_kv * group
        count, top = rng.choice([1, 2, 3, 8, 30, 200]), rng.choice([2, 20, 130, 300, 1500])
        if heads > 256 or count * top * heads > 400_000:
            continue
        lens_q = [rng.choice([0, 1, 1, 2, rng.randint(0, top)]) for _ in range(count)]
        lens_kv = [rng.choice([0, n, n, n + rng.randint(0, 300), rng.randint(0, 2 * top), n + rng.randint(0, 6000)])
                   for n in lens_q]
        prefix, causal = rng.choice([0, 0, 0, 1, 127, 128, 129, 777, 3000]), rng.random() < 0.6
        if prefix and causal:
            lens_kv = [max(a, b) for a, b in zip(lens_q, lens_kv)]
        pairs = sum(a * b for a, b in zip(lens_q, lens_kv)) + sum(lens_q) * prefix
        if pairs * heads > 3e8 or sum(lens_kv) > 300_000:
            continue
        starts = None
        if rng.random() < 0.5:
            starts, at = [0] * count, rng.randint(0, 50)
            for i in rng.sample(range(count), count):
                starts[i] = at
                at += lens_kv[i] + rng.randint(0, 40)
        return dict(lens_q=lens_q, lens_kv=lens_kv, heads=heads, heads_kv=heads_kv, causal=causal, starts=starts,
                    prefix=prefix, extra=rng.choice([0, 0, 3, 200]), spare=rng.choice([0, 5]),
                    nobody=math.nan if rng.random() < 0.7 else 1e30, by_head=rng.random() < 0.3,
                    loud=rng.choice([1, 1, 3]))


def run_attention(ops, case, gen):
    lens_q, lens_kv, prefix, starts = case["lens_q"], case["lens_kv"], case["prefix"], case["starts"]
    heads, heads_kv = case["heads"], case["heads_kv"]
    first = R.starts_of(lens_kv) if starts is None else starts
    rows = max([a + m for a, m in zip(first, lens_kv)], default=0)
    q = rand(gen, sum(lens_q) + case["extra"], heads, 128)
    q[sum(lens_q):] = case["nobody"]
    k, v = (torch.full((rows + case["extra"], heads_kv, 128), case["nobody"], device="cuda", dtype=torch.bfloat16)
            for _ in range(2))
    for at, m in zip(first, lens_kv):
        k[at:at + m], v[at:at + m] = rand(gen, m, heads_kv, 128) * case["loud"], rand(gen, m, heads_kv, 128)
    if case["by_head"]:
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=heads, heads_kv=heads_kv, causal=case["causal"], starts_kv=starts,
                             len_prefix=prefix)
    if prefix:
        kp, vp = (rand(gen, prefix + case["spare"], heads_kv, 128) for _ in range(2))
        call = lambda: ops.attention_shared_prefix(q, kp, vp, k, v, plan, return_lse=True)
        kp, vp = kp[:prefix], vp[:prefix]
        given = dict(k_prefix=kp, v_prefix=vp)
    else:
        call, given = lambda: ops.attention_packed(q, k, v, plan, return_lse=True), {}
    (o, lse), (again, lse_again) = call(), call()
    torch.cuda.synchronize()
    assert torch.equal(o, again) and torch.equal(lse, lse_again)
    assert (o[sum(lens_q):] == 0).all() and (lse[:, sum(lens_q):] == -math.inf).all()
    R.check_attention(o, lse, R.attention(q, k, v, lens_q, lens_kv, causal=case["causal"], starts=starts, **given))


def draw_rotation(rng):
    return dict(batch=rng.choice([0, 0, 1, 2, 5]), tokens=rng.choice([1, 2, 7, 33, 100, 1000, 4000]),
                heads=rng.randint(1, 40), heads_kv=rng.randint(0, 20), fused=rng.random() < 0.5,
                sections=rng.choice([(64,), (32,), (1,), (16, 24, 24), (24, 24), (5, 0, 9), (10, 20, 30, 4), (0, 64)]),
                weights=rng.choice([None, torch.bfloat16, torch.float32]), one_weight=rng.random() < 0.2,
                positions=rng.choice([torch.int32, torch.int64, torch.float32]), own_positions=rng.random() < 0.5,
                interleaved=rng.random() < 0.5, keys=rng.random() < 0.8, in_place=rng.random() < 0.3)


def run_rotation(ops, case, gen):
    batch, tokens, heads, heads_kv, sections = (case[n] for n in ("batch", "tokens", "heads", "heads_kv", "sections"))
    shape = (batch, tokens) if batch else (tokens,)
    rows = rand(gen, *shape, heads + heads_kv + 3, 128)
    q, k = rows[..., :heads, :], rows[..., heads + 1:heads + 1 + heads_kv, :]
    if not case["fused"]:
        q, k = q.contiguous(), k.contiguous()
    if not case["keys"]:
        k = None
    wq = wk = None
    if case["weights"] is not None:
        wq, wk = (rand(gen, 128, dtype=case["weights"]) for _ in range(2))
    if case["one_weight"] or k is None:
        wk = None
    pos_shape = (len(sections), batch, tokens) if batch and case["own_positions"] else (len(sections), tokens)
    pos = torch.randint(-1000, 100_000, pos_shape, generator=gen, device="cuda").to(case["positions"])
    f = torch.cat([10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float32) / max(n, 1)) for n in sections])
    before = [None if t is None else t.clone() for t in (q, k)]
    got = ops.qk_norm_rope(q, k, pos, f, sections=sections, q_weight=wq, k_weight=wk, eps=1e-6,
                           interleaved=case["interleaved"], out=(q, k) if case["in_place"] else None)
    torch.cuda.synchronize()
    for y, x, w in zip(got, before, (wq, wk)):
        if x is not None and x.numel():
            want, bound = R.rotate(x, w, pos, f, sections, eps=1e-6, interleaved=case["interleaved"])
            worst = ((y.double() - want).abs() - bound).max().item()
            assert worst <= 0.0, f"an element is {worst:.3e} beyond its bound"


def run(draw, run_case, seed, count):
    from b200_attention_b200 import _native, ops

    rng, gen = random.Random(seed), torch.Generator(device="cuda")
    gen.manual_seed(seed)
    for i in range(count):
        case = draw(rng)
        try:
            run_case(ops, case, gen)
        except AssertionError as e:
            raise AssertionError(f"case {i} of seed {seed}, {case}: {e}") from e
        _native.device_check()


@pytest.mark.parametrize("seed", range(1, 7))
def test_random_attention(native_built, seed):
    run(draw_attention, run_attention, seed, 10)


@pytest.mark.parametrize("seed", range(1, 5))
def test_random_rotation(native_built, seed):
    run(draw_rotation, run_rotation, seed, 20)


if __name__ == "__main__":
    count, seed = int(sys.argv[1]), int(sys.argv[2]) if len(sys.argv) > 2 else 100
    run(draw_attention, run_attention, seed, count)
    run(draw_rotation, run_rotation, seed, count)
    print(f"{count} attention and {count} rotation cases of seed {seed}: none beyond its bound")
