"""GPU tests of the serving operators together, in the order in which they are used: queries and keys normalised and
rotated, a whole batch of prompts attended, then new tokens against what is in the cache, with and without a shared
prefix, one plan for all layers of a step and one CUDA graph for all steps. Every stage is held to the plain 64-bit form
of its own inputs."""

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu
HEADS, HEADS_KV, EPS = 8, 2, 1e-6


@pytest.fixture(scope="module")
def ops(native_built):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    from b200_attention_b200 import _native, ops

    _native.lib()
    return ops


def settle():
    from b200_attention_b200 import _native

    torch.cuda.synchronize()
    _native.device_check()


def rand(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


class Layer:
    """Weights of one layer's norms, and its cache."""

    def __init__(self, seed, rows):
        self.q_weight, self.k_weight = 1 + 0.2 * rand(seed, 128), 1 + 0.2 * rand(seed + 1, 128)
        self.k = torch.full((rows, HEADS_KV, 128), float("nan"), device="cuda", dtype=torch.bfloat16)
        self.v = torch.full_like(self.k, float("nan"))


def freq():
    return 10000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float32) / 64)


def checked_rotation(ops, rows, layer, positions):
    """rows [tokens, HEADS + 2 * HEADS_KV, 128] of a fused projection; returns q, k, v."""
    q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + HEADS_KV], rows[:, HEADS + HEADS_KV:]
    qo, ko = ops.qk_norm_rope(q, k, positions, freq(), q_weight=layer.q_weight, k_weight=layer.k_weight, eps=EPS)
    for got, x, w in ((qo, q, layer.q_weight), (ko, k, layer.k_weight)):
        want, bound = R.rotate(x, w, positions[None], freq(), (64,), eps=EPS, interleaved=False)
        assert ((got.double() - want).abs() <= bound).all()
    return qo, ko, v


def test_prompts_then_tokens(ops):
    prompts = [300, 1, 129, 40]
    room = [n + 8 for n in prompts]
    starts = R.starts_of(room)
    layers = [Layer(10 * i, sum(room)) for i in range(2)]
    slots = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, prompts)]).cuda()
    positions = torch.cat([torch.arange(n) for n in prompts]).cuda()
    plan = ops.AttentionPlan(prompts, prompts, heads=HEADS, heads_kv=HEADS_KV, starts_kv=starts)
    for i, layer in enumerate(layers):
        q, k, v = checked_rotation(ops, rand(100 + i, sum(prompts), HEADS + 2 * HEADS_KV, 128), layer, positions)
        layer.k[slots], layer.v[slots] = k, v
        o, lse = ops.attention_packed(q, layer.k, layer.v, plan, return_lse=True)
        R.check_attention(o, lse, R.attention(q, layer.k, layer.v, prompts, prompts, causal=True, starts=starts))
    lens = list(prompts)
    plan = ops.AttentionPlan([1] * 4, [n + 1 for n in lens], heads=HEADS, heads_kv=HEADS_KV, starts_kv=starts)
    for step in range(4):
        lens = [n + 1 for n in lens]
        plan.update([1] * 4, lens, starts_kv=starts)
        last = torch.tensor([a + n - 1 for a, n in zip(starts, lens)], device="cuda")
        positions = torch.tensor([n - 1 for n in lens], device="cuda")
        for i, layer in enumerate(layers):
            q, k, v = checked_rotation(ops, rand(200 + 10 * step + i, 4, HEADS + 2 * HEADS_KV, 128), layer, positions)
            layer.k[last], layer.v[last] = k, v
            o, lse = ops.attention_packed(q, layer.k, layer.v, plan, return_lse=True)
            R.check_attention(o, lse, R.attention(q, layer.k, layer.v, [1] * 4, lens, causal=True, starts=starts))
    settle()


def test_tokens_one_by_one_agree_with_the_whole_prompt(ops):
    """The last token of every length against a cache that goes on (with rows that it must not see) gives the rows of the
    whole prompt's call: both are within their bound of the same exact result."""
    n = 140
    q, k, v = rand(1, n, HEADS, 128), rand(2, n, HEADS_KV, 128), rand(3, n, HEADS_KV, 128)
    whole = ops.attention_packed(q, k, v, ops.AttentionPlan([n], [n], heads=HEADS, heads_kv=HEADS_KV))
    lens = list(range(1, n + 1))
    single = ops.attention_packed(q, k, v, ops.AttentionPlan([1] * n, lens, heads=HEADS, heads_kv=HEADS_KV,
                                                             starts_kv=[0] * n))
    settle()
    ref = R.attention(q, k, v, [n], [n], causal=True)
    R.check_attention(whole, None, ref)
    R.check_attention(single, None, ref)


def test_a_prefix_agrees_with_its_keys_in_every_cache(ops):
    prefix, own = 700, [5, 130, 1, 64]
    lens_q = [1, 3, 1, 2]
    q = rand(1, sum(lens_q), HEADS, 128)
    kp, vp = rand(2, prefix, HEADS_KV, 128), rand(3, prefix, HEADS_KV, 128)
    k, v = rand(4, sum(own), HEADS_KV, 128), rand(5, sum(own), HEADS_KV, 128)
    a, a_lse = ops.attention_shared_prefix(q, kp, vp, k, v, ops.AttentionPlan(lens_q, own, heads=HEADS, heads_kv=HEADS_KV,
                                                                              len_prefix=prefix), return_lse=True)
    full = [torch.cat([torch.cat([p, t[s:s + m]]) for s, m in zip(R.starts_of(own), own)]) for p, t in ((kp, k), (vp, v))]
    b, b_lse = ops.attention_packed(q, *full, ops.AttentionPlan(lens_q, [prefix + m for m in own], heads=HEADS,
                                                                heads_kv=HEADS_KV), return_lse=True)
    settle()
    ref = R.attention(q, k, v, lens_q, own, causal=True, k_prefix=kp, v_prefix=vp)
    R.check_attention(a, a_lse, ref)
    R.check_attention(b, b_lse, ref)


def test_one_graph_for_all_steps(ops):
    """Rotation and attention behind a shared prefix, captured once; plan, positions and rows change between replays."""
    count, prefix, room = 5, 300, 64
    layer = Layer(3, count * room)
    starts = [i * room for i in range(count)]
    kp, vp = rand(7, prefix, HEADS_KV, 128), rand(8, prefix, HEADS_KV, 128)
    lens = [3, 17, 1, 30, 8]
    for a, n in zip(starts, lens):
        layer.k[a:a + n], layer.v[a:a + n] = rand(20 + a, n, HEADS_KV, 128), rand(21 + a, n, HEADS_KV, 128)
    plan = ops.AttentionPlan([1] * count, [n + 1 for n in lens], heads=HEADS, heads_kv=HEADS_KV, starts_kv=starts,
                             len_prefix=prefix)
    rows = rand(30, count, HEADS + 2 * HEADS_KV, 128)
    positions = torch.tensor([prefix + n for n in lens], device="cuda")
    last = torch.tensor([a + n for a, n in zip(starts, lens)], device="cuda")
    f = freq()

    def step():
        q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + HEADS_KV], rows[:, HEADS + HEADS_KV:]
        q, k = ops.qk_norm_rope(q, k, positions, f, q_weight=layer.q_weight, k_weight=layer.k_weight, eps=EPS)
        layer.k.index_copy_(0, last, k)
        layer.v.index_copy_(0, last, v)
        return q, ops.attention_shared_prefix(q, kp, vp, layer.k, layer.v, plan)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, o = step()
    for i in range(4):
        lens = [n + 1 for n in lens]
        plan.update([1] * count, lens, starts_kv=starts)
        rows.copy_(rand(40 + i, count, HEADS + 2 * HEADS_KV, 128))
        positions.copy_(torch.tensor([prefix + n - 1 for n in lens]))
        last.copy_(torch.tensor([a + n - 1 for a, n in zip(starts, lens)]))
        graph.replay()
        settle()
        want, bound = R.rotate(rows[:, :HEADS], layer.q_weight, positions[None], f, (64,), eps=EPS, interleaved=False)
        assert ((q.double() - want).abs() <= bound).all()
        R.check_attention(o, None, R.attention(q, layer.k, layer.v, [1] * count, lens, causal=True, starts=starts,
                                               k_prefix=kp, v_prefix=vp))
    del graph


def test_attention_callable_with_norm_and_rotation(ops):
    """The video model's callable on raw projections: time, height and width positions, norm per head."""
    from b200_attention_b200.backend import B200Attention

    b, (t, h, w), heads = 2, (3, 5, 9), 3
    n = t * h * w
    i = torch.arange(n, device="cuda")
    positions = torch.stack([i // (h * w), i // w % h, i % w])
    sections = (16, 24, 24)
    f = torch.cat([10000.0 ** (-torch.arange(m, device="cuda", dtype=torch.float32) / m) for m in sections])
    wq, wk = 1 + 0.2 * rand(1, 128), 1 + 0.2 * rand(2, 128)
    qk = ops.QkNormRope(positions, f, sections=sections, q_weight=wq, k_weight=wk, interleaved=True)
    q, k, v = (rand(3 + j, b, n, heads * 128) for j in range(3))
    out = B200Attention(qk=qk)(q, k, v, heads)
    q4, k4 = qk(q.view(b, n, heads, 128), k.view(b, n, heads, 128))
    settle()
    for got, x, wt in ((q4, q, wq), (k4, k, wk)):
        want, bound = R.rotate(x.view(b, n, heads, 128), wt, positions, f, sections, eps=1e-6, interleaved=True)
        assert ((got.double() - want).abs() <= bound).all()
    flat = [x.reshape(b * n, heads, 128) for x in (q4, k4, v.view(b, n, heads, 128))]
    R.check_attention(out.view(b * n, heads, 128), None, R.attention(*flat, [n] * b, [n] * b, causal=False))
    with pytest.raises(RuntimeError, match="disagree"):
        B200Attention(qk=qk)(q, k[:, :7], v[:, :7], heads)   # cross-attention: its keys have no such positions
