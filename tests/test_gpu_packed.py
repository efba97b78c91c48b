"""GPU tests of attention over packed sequences and over a shared prefix, against the plain 64-bit forms."""

import math

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu


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


def make(lens_q, lens_kv, heads, heads_kv, *, seed=0, starts=None, prefix=0, extra=0):
    """q, k, v (and prefix); rows of k and v that belong to no sequence, and rows of q behind the last, hold NaN."""
    rows_kv = sum(lens_kv) if starts is None else max(a + m for a, m in zip(starts, lens_kv))
    q = rand(seed, sum(lens_q) + extra, heads, 128)
    q[sum(lens_q):] = math.nan
    k, v = (torch.full((rows_kv + extra, heads_kv, 128), math.nan, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for at, m in zip(R.starts_of(lens_kv) if starts is None else starts, lens_kv):
        k[at:at + m], v[at:at + m] = rand(seed + 1 + at, m, heads_kv, 128), rand(seed + 2 + at, m, heads_kv, 128)
    pre = (rand(seed + 3, prefix, heads_kv, 128), rand(seed + 4, prefix, heads_kv, 128)) if prefix else (None, None)
    return q, k, v, *pre


def run_case(ops, lens_q, lens_kv, heads, heads_kv, *, causal=True, starts=None, prefix=0, extra=0, scale=None, seed=0):
    q, k, v, kp, vp = make(lens_q, lens_kv, heads, heads_kv, seed=seed, starts=starts, prefix=prefix, extra=extra)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=heads, heads_kv=heads_kv, causal=causal, starts_kv=starts,
                             len_prefix=prefix)
    kw = dict(return_lse=True, softmax_scale=scale or 0.0)
    if prefix:
        o, lse = ops.attention_shared_prefix(q, kp, vp, k, v, plan, **kw)
    else:
        o, lse = ops.attention_packed(q, k, v, plan, **kw)
    settle()
    ref = R.attention(q, k, v, lens_q, lens_kv, causal=causal, starts=starts, k_prefix=kp, v_prefix=vp, scale=scale)
    R.check_attention(o, lse, ref)
    rows = sum(lens_q)
    assert (o[rows:] == 0).all() and (lse[:, rows:] == -math.inf).all()
    return o, lse


PACKED = [
    # lens_q, lens_kv, heads, heads_kv, causal
    ([1], [1], 1, 1, True),
    ([128], [128], 1, 1, True),
    ([129], [129], 2, 2, True),                        # a second Q tile of one row
    ([256, 256], [256, 256], 2, 2, True),
    ([257], [257], 1, 1, False),                       # a second item of one row
    ([17, 1, 64, 129, 5], [17, 1, 64, 129, 5], 8, 2, True),
    ([17, 1, 64, 129, 5], [17, 1, 64, 129, 5], 8, 2, False),
    ([200, 1, 129, 7], [5, 1, 100, 0], 4, 4, True),    # rows, tiles and sequences that see nothing
    ([0, 5, 0, 3], [7, 5, 0, 0], 4, 2, False),         # empty sequences among others
    ([3], [0], 4, 2, True),                            # no key at all
    ([100, 60], [1000, 2000], 6, 2, True),             # chunks with history, 42 tokens to a tile
    ([70, 33], [700, 33], 5, 1, True),                 # 25 tokens to a tile
    ([40], [300], 128, 1, True),                       # one token to a tile
    ([9], [500], 96, 1, False),                        # one token to a tile, a quarter of it idle
    ([700, 1300, 64], [700, 1300, 64], 12, 12, False),
    ([1], [9000], 8, 1, True),                         # one token, cut into pieces
    ([1] * 20, [1 + 150 * i for i in range(20)], 16, 2, True),
    ([4, 1, 2], [4000, 5000, 130], 8, 8, True),        # a few tokens each
    ([2048, 1, 900], [2048, 3500, 900], 16, 4, True),  # a prompt beside a decode step
]


@pytest.mark.parametrize("case", PACKED, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-{c[2]}-{c[3]}-{c[4]}".replace(" ", ""))
def test_packed(ops, case):
    lens_q, lens_kv, heads, heads_kv, causal = case
    run_case(ops, lens_q, lens_kv, heads, heads_kv, causal=causal)


@pytest.mark.parametrize("prefix, lens_q, lens_kv, heads, heads_kv, causal", [
    (1, [1], [1], 1, 1, True),
    (128, [1, 1], [1, 128], 4, 2, True),
    (1000, [1, 1, 1, 1], [1, 37, 64, 12], 16, 4, True),
    (777, [1, 4, 2, 1], [300, 4, 9, 129], 6, 2, True),   # several tokens each, mask among them
    (5000, [1] * 70, [1 + 5 * i for i in range(70)], 8, 2, True),   # two blocks of tokens for the prefix
    (300, [150, 0, 130], [150, 0, 200], 8, 4, True),     # blocks across sequences
    (129, [2, 3], [0, 0], 4, 4, False),                  # the prefix alone
    (640, [3, 1], [5, 0], 2, 2, False),
])
def test_shared_prefix(ops, prefix, lens_q, lens_kv, heads, heads_kv, causal):
    run_case(ops, lens_q, lens_kv, heads, heads_kv, causal=causal, prefix=prefix)


@pytest.mark.parametrize("prefix", [0, 513])
def test_rows_outside_the_sequences_have_no_influence(ops, prefix):
    """A cache with room between the sequences and in another order than theirs; all that is not theirs is NaN, and so
    are the rows of q behind the last one."""
    lens_q, lens_kv, starts = [1, 3, 1, 140], [100, 257, 1, 140], [700, 50, 500, 512]
    run_case(ops, lens_q, lens_kv, 8, 4, starts=starts, prefix=prefix, extra=9)


def test_sequences_may_share_keys(ops):
    run_case(ops, [1, 5], [300, 305], 4, 2, starts=[0, 0])


@pytest.mark.parametrize("scale", [0.02, 0.5])
def test_softmax_scale(ops, scale):
    run_case(ops, [100, 1], [333, 450], 4, 2, scale=scale)


def test_scores_that_grow_along_the_keys(ops):
    """The rows' reference maximum has to move far, many times, in every tile of a masked and a split row."""
    lens_q, lens_kv = [130, 1], [900, 6000]
    q, k, v, _, _ = make(lens_q, lens_kv, 4, 2, seed=5)
    for at, m in zip(R.starts_of(lens_kv), lens_kv):
        k[at:at + m] *= torch.linspace(0.1, 30.0, m, device="cuda", dtype=torch.bfloat16)[:, None, None]
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=4, heads_kv=2)
    o, lse = ops.attention_packed(q, k, v, plan, return_lse=True)
    settle()
    o_ref, lse_ref, spread = R.attention(q, k, v, lens_q, lens_kv, causal=True)
    # scores up to 400 here: in 32 bits they are off by up to 400 * 128 * 2^-24 = 2^-8.4 in the worst case, which moves a
    # probability by as much, relative, and numerator and row sum both
    bound = (R.HALF_STEP + 2 * 2.0 ** -8.4) * spread + R.HALF_STEP * (o_ref.abs() + 2.0 ** -6 * spread)
    assert ((o.double() - o_ref).abs() <= bound).all()
    assert ((lse.double() - lse_ref).abs() <= 2.0 ** -8.4 + 2.0 ** -12).all()


def test_values_that_are_not_finite_stay_in_their_sequence(ops):
    """An infinity or NaN in one request's keys or values reaches that request's rows and no other's."""
    lens_q, lens_kv = [40, 50, 1, 1], [40, 50, 300, 200]
    q, k, v, _, _ = make(lens_q, lens_kv, 4, 2)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=4, heads_kv=2)
    clean = ops.attention_packed(q, k, v, plan)
    k[45], v[47, :, 3], k[391], v[395] = math.nan, math.inf, math.inf, math.nan   # sequences 1 and 3
    spoilt = ops.attention_packed(q, k, v, plan)
    settle()
    for rows in (slice(0, 40), slice(90, 91)):
        assert torch.equal(spoilt[rows], clean[rows])
    assert torch.isnan(spoilt[89]).any() and torch.isnan(spoilt[91]).any()


def test_strided_operands(ops):
    """q, k and v cut out of fused rows, o into a wider buffer, heads before rows."""
    lens_q, lens_kv = [150, 1, 30], [150, 1, 30]
    rows = rand(1, 181, 8 + 2 + 2, 128)
    q, k, v = rows[:, :8], rows[:, 8:10], rows[:, 10:]
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2)
    want = ops.attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), plan)
    wide = torch.full((181, 10, 256), 7.0, device="cuda", dtype=torch.bfloat16)
    got = ops.attention_packed(q, k, v, plan, out=wide[:, 1:9, :128])
    odd = torch.full((181, 8, 136), 7.0, device="cuda", dtype=torch.bfloat16)  # rows on multiples of 16 bytes, not of 32
    ops.attention_packed(q, k, v, plan, out=odd[:, :, 8:])
    by_head = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    other = ops.attention_packed(*by_head, plan)
    settle()
    R.check_attention(want, None, R.attention(q, k, v, lens_q, lens_kv, causal=True))
    assert torch.equal(got, want) and torch.equal(other, want)
    assert torch.equal(odd[:, :, 8:], want) and (odd[:, :, :8] == 7).all()
    assert (wide[:, 0] == 7).all() and (wide[:, 9] == 7).all() and (wide[:, :, 128:] == 7).all()


def test_result_in_the_place_of_q(ops):
    """out may be q itself: whole items, cut ones, and rows joined with a prefix."""
    for lens_q, lens_kv, prefix in [([300, 1, 40], [300, 9, 40], 0), ([1, 2], [9000, 5000], 0), ([1] * 9, [50] * 9, 700)]:
        q, k, v, kp, vp = make(lens_q, lens_kv, 8, 2, prefix=prefix)
        plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2, len_prefix=prefix)
        call = lambda out: (ops.attention_shared_prefix(q, kp, vp, k, v, plan, out=out) if prefix
                            else ops.attention_packed(q, k, v, plan, out=out))
        want = call(torch.empty_like(q))
        got = call(q)
        settle()
        assert got is q or got.data_ptr() == q.data_ptr()
        assert torch.equal(q, want)


def test_a_cache_whose_offsets_pass_32_bits(ops):
    """Sequences at the end of a cache of 2.3e9 elements (4.6 GB each for k and v)."""
    heads_kv, rows = 8, 2_250_000
    lens_q, lens_kv = [1, 20], [700, 333]
    starts = [rows - 400 - 700, rows - 333]
    k, v = (torch.empty(rows, heads_kv, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for t in (k, v):
        t[:1000] = math.nan
        t[rows - 2000:] = rand(5 if t is k else 6, 2000, heads_kv, 128)
    assert starts[0] * heads_kv * 128 > 2**31
    q = rand(3, sum(lens_q), 16, 128)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=16, heads_kv=heads_kv, starts_kv=starts)
    o, lse = ops.attention_packed(q, k, v, plan, return_lse=True)
    settle()
    R.check_attention(o, lse, R.attention(q, k, v, lens_q, lens_kv, causal=True, starts=starts))


def test_rows_behind_the_last_sequence_keep_what_they_hold(ops):
    q, k, v, kp, vp = make([3, 2], [9, 2], 4, 2, extra=5, prefix=20)
    out = torch.full_like(q, 3.0)
    plan = ops.AttentionPlan([3, 2], [9, 2], heads=4, heads_kv=2, len_prefix=20)
    ops.attention_shared_prefix(q, kp, vp, k, v, plan, out=out)
    settle()
    assert (out[5:] == 3).all() and torch.isfinite(out[:5]).all()


def test_a_row_that_sees_one_key_is_its_value(ops):
    """One probability of exactly 1: nothing is rounded on the way, whatever the score."""
    lens = [1, 7, 1, 300, 64]
    q, k, v, _, _ = make(lens, lens, 8, 2)
    plan = ops.AttentionPlan(lens, lens, heads=8, heads_kv=2)
    o = ops.attention_packed(q * 3, k, v, plan)
    settle()
    first = R.starts_of(lens)
    assert torch.equal(o[first], v[first].repeat_interleave(4, dim=1))


def test_results_repeat(ops):
    lens_q, lens_kv = [1] * 9 + [64], [1 + 700 * i for i in range(9)] + [64]
    q, k, v, kp, vp = make(lens_q, lens_kv, 16, 4, prefix=3500)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=16, heads_kv=4, len_prefix=3500, causal=False)
    first = ops.attention_shared_prefix(q, kp, vp, k, v, plan, return_lse=True)
    for _ in range(5):
        again = ops.attention_shared_prefix(q, kp, vp, k, v, plan, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    settle()


def test_many_launches_in_a_row(ops):
    """Back to back, pieces of every kind on every CTA; no wait may run out."""
    lens_q = [1, 300, 5, 1, 77, 128, 1, 1] * 6
    lens_kv = [900, 300, 5, 129, 500, 128, 2000, 1] * 6
    q, k, v, _, _ = make(lens_q, lens_kv, 12, 4)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=12, heads_kv=4)
    first = ops.attention_packed(q, k, v, plan)
    for _ in range(200):
        again = ops.attention_packed(q, k, v, plan)
    settle()
    assert torch.equal(first, again)
    R.check_attention(first, None, R.attention(q, k, v, lens_q, lens_kv, causal=True))


def test_more_pieces_than_a_cta_keeps_at_hand(ops):
    """Thousands of tiny sequences: the later pieces of a CTA come from the table in memory."""
    lens = [1 + i % 3 for i in range(9000)]
    run_case(ops, lens, lens, 4, 4)


@pytest.mark.parametrize("lens_q, lens_kv, prefix", [([1, 40, 300, 5], [700, 40, 900, 131], 0), ([1] * 40, [300] * 40, 0), ([70, 1], [70, 130], 600)])
def test_both_builds_of_the_kernel_take_every_plan(ops, lens_q, lens_kv, prefix):
    """Whichever the plan asks for (by its wide pieces): a captured call keeps the one that it was captured with."""
    q, k, v, kp, vp = make(lens_q, lens_kv, 8, 2, prefix=prefix)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2, len_prefix=prefix)
    wide = plan._now[-1]
    assert (wide > 0) == (max(lens_q) > 32 or prefix > 0)  # 32 tokens x 4 heads of a group fill a Q tile
    results = []
    for hint in (wide, 0, 1):
        plan._now = (*plan._now[:-1], hint)
        if prefix:
            results.append(ops.attention_shared_prefix(q, kp, vp, k, v, plan, return_lse=True))
        else:
            results.append(ops.attention_packed(q, k, v, plan, return_lse=True))
        settle()
    R.check_attention(*results[0], R.attention(q, k, v, lens_q, lens_kv, causal=True, k_prefix=kp, v_prefix=vp))
    for o, lse in results[1:]:
        assert torch.equal(o, results[0][0]) and torch.equal(lse, results[0][1])


def test_agrees_with_the_rectangular_call(ops):
    b, n = 3, 640
    q, k, v = rand(1, b * n, 8, 128), rand(2, b * n, 2, 128), rand(3, b * n, 2, 128)
    plan = ops.AttentionPlan([n] * b, [n] * b, heads=8, heads_kv=2)
    o, lse = ops.attention_packed(q, k, v, plan, return_lse=True)
    shape = lambda t: t.view(b, n, -1, 128)
    o2, lse2 = ops.attention(shape(q), shape(k), shape(v), layout="bshd", causal=True, return_lse=True)
    settle()
    # each is within 2^-7 of the exact result, relative to values below 4 here
    assert (shape(o).float() - o2.float()).abs().max() <= 2 * 4 * 2.0 ** -7
    assert (lse.view(8, b, n).transpose(0, 1) - lse2).abs().max() <= 2.0 ** -11


def test_two_streams_and_another_thread_of_work(ops):
    lens_q, lens_kv = [1] * 6, [4000 + 100 * i for i in range(6)]
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2)
    sets = [make(lens_q, lens_kv, 8, 2, seed=s)[:3] for s in (0, 50)]
    want = [ops.attention_packed(*t, plan) for t in sets]
    settle()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            got[i].append(ops.attention_packed(*sets[i], plan, stream=s))
    settle()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_shared_prefix_on_another_stream(ops):
    lens_q, lens_kv = [1, 2, 1], [50, 130, 9]
    q, k, v, kp, vp = make(lens_q, lens_kv, 8, 2, prefix=2000)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2, len_prefix=2000)
    want, want_lse = ops.attention_shared_prefix(q, kp, vp, k, v, plan, return_lse=True)
    settle()
    s = torch.cuda.Stream()
    late = torch.empty_like(q)
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)  # what the call reads is only written now
    got, lse = ops.attention_shared_prefix(late, kp, vp, k, v, plan, return_lse=True, stream=s)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    settle()


def test_a_plan_may_go_while_another_stream_uses_it(ops):
    lens_q, lens_kv = [1, 2, 1], [50, 130, 9]
    q, k, v, _, _ = make(lens_q, lens_kv, 8, 2)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2)
    want = ops.attention_packed(q, k, v, plan)
    settle()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(40_000_000)
    got = ops.attention_packed(q, k, v, plan, stream=s)
    place, size = plan._table.data_ptr(), plan._table.numel()
    del plan
    others = [torch.zeros(size, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not s.query(), "the call was to be waiting still"
    assert place not in [t.data_ptr() for t in others]
    s.synchronize()
    assert torch.equal(got, want)
    settle()


def test_given_outputs_count_as_changed(ops):
    q, k, v, _, _ = make([3], [5], 4, 2)
    plan = ops.AttentionPlan([3], [5], heads=4, heads_kv=2)
    w = torch.ones(4, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    saved = (q * w).sum()  # keeps q for the gradient of w
    ops.attention_packed(q, k, v, plan, out=q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    with torch.inference_mode():
        o = torch.empty_like(q)
        ops.attention_packed(q, k, v, plan, out=o)
    settle()


def test_captured_call_follows_an_updated_plan(ops):
    q, k, v, kp, vp = make([1] * 4, [600] * 4, 8, 2, prefix=700)
    starts = [0, 600, 1200, 1800]
    lens = [100, 250, 3, 400]
    plan = ops.AttentionPlan([1] * 4, lens, heads=8, heads_kv=2, starts_kv=starts, len_prefix=700)
    out = torch.empty_like(q)
    ops.attention_shared_prefix(q, kp, vp, k, v, plan, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_shared_prefix(q, kp, vp, k, v, plan, out=out)
    for step in range(3):
        now = [n + 60 * step for n in lens]
        plan.update([1] * 4, now, starts_kv=starts)
        out.fill_(math.nan)
        graph.replay()
        settle()
        ref = R.attention(q, k, v, [1] * 4, now, causal=True, starts=starts, k_prefix=kp, v_prefix=vp)
        R.check_attention(out, None, ref)
    with pytest.raises(RuntimeError, match="do not fit"):
        plan.update([2] * 4, lens, starts_kv=starts)             # more rows than the captured q has
    with pytest.raises(RuntimeError, match="do not fit"):
        plan.update([1] * 4, lens, starts_kv=[0, 600, 1200, 2001])  # past the captured k
    del graph


def test_two_graphs_of_one_plan_overlap(ops):
    lens_q, lens_kv = [1] * 5, [5000] * 5
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=1)
    sets = [make(lens_q, lens_kv, 8, 1, seed=s)[:3] for s in (0, 90)]
    want = [ops.attention_packed(*t, plan) for t in sets]
    settle()
    graphs, outs = [], []
    for t in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.attention_packed(*t, plan))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    settle()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    del graphs


def test_a_graph_outlives_its_plan(ops):
    """The table that a captured call reads stays, and so does the memory that its replays need."""
    import gc

    lens_q, lens_kv = [1, 40], [3000, 40]
    q, k, v, _, _ = make(lens_q, lens_kv, 8, 2)
    plan = ops.AttentionPlan(lens_q, lens_kv, heads=8, heads_kv=2)
    want = ops.attention_packed(q, k, v, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.attention_packed(q, k, v, plan)
    del plan
    gc.collect()
    torch.cuda.empty_cache()
    noise = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (1000, 20000, 30000, 100000)]
    graph.replay()
    settle()
    assert torch.equal(got, want)
    del graph, noise


def test_plans_and_updates_are_refused_in_a_capture(ops):
    plan = ops.AttentionPlan([1], [5], heads=2)
    x = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="captured"):
            ops.AttentionPlan([1], [5], heads=2)
        with pytest.raises(RuntimeError, match="captured"):
            plan.update([1], [6])
    graph.replay()
    settle()
    assert x.item() == 1
    del graph


def test_update_in_eager_use(ops):
    plan = ops.AttentionPlan([1], [5], heads=2)
    for lens_q, lens_kv in [([1], [700]), ([300, 2], [300, 9]), ([1] * 50, [4000] * 50)]:
        plan.update(lens_q, lens_kv)
        q, k, v, _, _ = make(lens_q, lens_kv, 2, 2)
        o = ops.attention_packed(q, k, v, plan)
        settle()
        R.check_attention(o, None, R.attention(q, k, v, lens_q, lens_kv, causal=True))


def test_refusals(ops):
    q, k, v, kp, vp = make([3], [9], 4, 2, prefix=20)
    plan = ops.AttentionPlan([3], [9], heads=4, heads_kv=2)
    shared = ops.AttentionPlan([3], [9], heads=4, heads_kv=2, len_prefix=20)
    bad = [
        lambda: ops.attention_packed(q.float(), k, v, plan),
        lambda: ops.attention_packed(q[:2], k, v, plan),
        lambda: ops.attention_packed(q, k[:8], v[:8], plan),
        lambda: ops.attention_packed(q, k, v[:8], plan),
        lambda: ops.attention_packed(q[:, :2], k, v, plan),
        lambda: ops.attention_packed(q, k[:, :1], v[:, :1], plan),
        lambda: ops.attention_packed(q[..., :64], k, v, plan),
        lambda: ops.attention_packed(q[None], k, v, plan),
        lambda: ops.attention_packed(q.cpu(), k, v, plan),
        lambda: ops.attention_packed(q, k, v, shared),
        lambda: ops.attention_packed(q, k, v, plan, out=torch.empty_like(k)),
        lambda: ops.attention_packed(q.clone().requires_grad_(), k, v, plan),
        lambda: ops.attention_packed(q.transpose(0, 2).contiguous().transpose(0, 2), k, v, plan),
        lambda: ops.attention_shared_prefix(q, kp, vp, k, v, plan),
        lambda: ops.attention_shared_prefix(q, kp[:19], vp, k, v, shared),
        lambda: ops.attention_shared_prefix(q, kp, vp[:, :1], k, v, shared),
        lambda: ops.attention_packed(torch.zeros(3 * 512 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(3, 4, 128), k, v, plan),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")
    with torch.no_grad():
        ops.attention_packed(q.clone().requires_grad_(), k, v, plan)
    with pytest.raises(RuntimeError, match="host integers"):
        ops.AttentionPlan(torch.tensor([3], device="cuda"), [9], heads=2)
    settle()
