"""GPU tests of the norm and rotation of queries and keys, against the plain 64-bit form."""

import math

import pytest
import torch

from tests import packed_reference as R

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def ops(native_built):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    from b200_attention_b200 import _native, ops

    _native.lib()
    return ops


def rand(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def freqs(sections):
    return torch.cat([10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float32) / max(n, 1)) for n in sections])


def check(got, x, weight, positions, inv_freq, sections, interleaved, eps=EPS):
    want, bound = R.rotate(x, weight, positions, inv_freq, sections, eps=eps, interleaved=interleaved)
    worst = ((got.double() - want).abs() - bound).max().item()
    assert worst <= 0.0, f"an element is {worst:.3e} beyond its bound"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape, heads, heads_kv, sections, weights", [
    ((1,), 1, 1, (64,), None),
    ((1,), 3, 2, (64,), torch.bfloat16),
    ((3,), 32, 8, (64,), torch.float32),
    ((2, 5), 12, 12, (16, 24, 24), torch.bfloat16),
    ((1537,), 20, 4, (24, 24), None),
    ((3, 333), 5, 1, (1, 0, 2, 5), torch.bfloat16),
    ((9000,), 7, 7, (10, 21, 30), torch.bfloat16),
    ((2, 4000), 40, 8, (64,), torch.float32),
])
def test_rotation(ops, shape, heads, heads_kv, sections, weights, interleaved):
    q, k = rand(1, *shape, heads, 128), rand(2, *shape, heads_kv, 128) * 3
    wq = wk = None
    if weights is not None:
        wq, wk = 1 + 0.3 * rand(3, 128, dtype=weights), 1 + 0.3 * rand(4, 128, dtype=weights)
    pos = torch.randint(-5, 5000, (len(sections), shape[-1]), device="cuda")
    f = freqs(sections)
    qo, ko = ops.qk_norm_rope(q, k, pos, f, sections=sections, q_weight=wq, k_weight=wk, interleaved=interleaved)
    torch.cuda.synchronize()
    check(qo, q, wq, pos, f, sections, interleaved)
    check(ko, k, wk, pos, f, sections, interleaved)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32])
def test_far_positions_and_position_types(ops, dtype):
    q, k = rand(1, 64, 2, 128), rand(2, 64, 1, 128)
    pos = (torch.arange(64, device="cuda") * 16 + (2**24 - 1024)).to(dtype)
    f = freqs((64,))
    qo, ko = ops.qk_norm_rope(q, k, pos, f)
    torch.cuda.synchronize()
    check(qo, q, None, pos[None], f, (64,), False)
    check(ko, k, None, pos[None], f, (64,), False)


def test_fractional_positions_of_a_batch(ops):
    q = rand(1, 3, 50, 4, 128)
    pos = rand(2, 2, 3, 50, dtype=torch.float32) * 100
    f = freqs((30, 34))
    qo, none = ops.qk_norm_rope(q, None, pos, f, sections=(30, 34), q_weight=rand(3, 128))
    torch.cuda.synchronize()
    assert none is None
    check(qo, q, rand(3, 128), pos, f, (30, 34), False)


@pytest.mark.parametrize("norm", [False, True])
def test_one_weight_only(ops, norm):
    q, k, w, pos, f = rand(1, 9, 4, 128), rand(2, 9, 2, 128), rand(3, 128), torch.arange(9, device="cuda"), freqs((64,))
    qo, ko = ops.qk_norm_rope(q, k, pos, f, q_weight=w if norm else None, k_weight=None if norm else w)
    torch.cuda.synchronize()
    check(qo, q, w if norm else None, pos[None], f, (64,), False)
    check(ko, k, None if norm else w, pos[None], f, (64,), False)


@pytest.mark.parametrize("eps", [0.0, 1e-6, 0.5])
def test_small_and_zero_rows(ops, eps):
    q = rand(1, 40, 2, 128) * 1e-4
    w, pos, f = rand(3, 128), torch.arange(40, device="cuda"), freqs((64,))
    zero = torch.zeros_like(q)
    qo, zo = ops.qk_norm_rope(q, zero, pos, f, q_weight=w, k_weight=w, eps=eps)
    torch.cuda.synchronize()
    check(qo, q, w, pos[None], f, (64,), False, eps=eps)
    assert torch.isnan(zo).all() if eps == 0 else (zo == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_fused_rows_in_place(ops, interleaved):
    """q and k cut out of the rows of one projection and written back to their places; v is left alone."""
    rows = rand(1, 2, 77, 6 + 2 + 2, 128)
    before = rows.clone()
    q, k = rows[:, :, :6], rows[:, :, 6:8]
    pos, f, w = torch.arange(77, device="cuda"), freqs((64,)), rand(3, 128)
    qo, ko = ops.qk_norm_rope(q, k, pos, f, q_weight=w, k_weight=w, interleaved=interleaved, out=(q, k))
    torch.cuda.synchronize()
    assert qo is q and ko is k and torch.equal(rows[:, :, 8:], before[:, :, 8:])
    check(q, before[:, :, :6], w, pos[None], f, (64,), interleaved)
    check(k, before[:, :, 6:8], w, pos[None], f, (64,), interleaved)


def test_strides_streams_and_graphs(ops):
    """Heads before tokens, an output inside a wider buffer, another stream, a captured call."""
    q = rand(1, 4, 100, 128).transpose(0, 1)                  # [tokens, heads, 128], heads outermost
    k = rand(2, 100, 3, 256)[:, :, 64:192]
    pos, f = torch.arange(100, device="cuda"), freqs((64,))
    wide = torch.full((100, 9, 128), 5.0, device="cuda", dtype=torch.bfloat16)
    out = (wide[:, 1:5], wide[:, 5:8])
    want = ops.qk_norm_rope(q, k, pos, f)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ops.qk_norm_rope(q, k, pos, f, out=out, stream=s)
    torch.cuda.synchronize()
    check(want[0], q, None, pos[None], f, (64,), False)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert (wide[:, 0] == 5).all() and (wide[:, 8] == 5).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.qk_norm_rope(q, k, pos, f)
    pos += 7
    graph.replay()
    torch.cuda.synchronize()
    check(got[0], q, None, pos[None], f, (64,), False)
    del graph


def test_offsets_past_32_bits(ops):
    """2.3e9 elements: the last tokens' rows begin behind 2^31."""
    tokens, heads = 70_001, 256
    q = torch.empty(tokens, heads, 128, device="cuda", dtype=torch.bfloat16)
    q[-8:] = rand(1, 8, heads, 128)
    q[:8] = rand(2, 8, heads, 128)
    assert (tokens - 8) * heads * 128 > 2**31
    pos, f = torch.arange(tokens, device="cuda"), freqs((64,))
    qo, _ = ops.qk_norm_rope(q, None, pos, f)
    torch.cuda.synchronize()
    check(qo[-8:], q[-8:], None, pos[None, -8:], f, (64,), False)
    check(qo[:8], q[:8], None, pos[None, :8], f, (64,), False)


def test_values_that_are_not_finite_stay_in_their_head(ops):
    q = rand(1, 5, 4, 128)
    q[2, 1, 7], q[3, 0, 100] = math.nan, math.inf
    pos, f, w = torch.arange(5, device="cuda"), freqs((64,)), rand(3, 128)
    qo, _ = ops.qk_norm_rope(q, None, pos, f, q_weight=w)
    torch.cuda.synchronize()
    bad = torch.zeros(5, 4, dtype=torch.bool, device="cuda")
    bad[2, 1] = bad[3, 0] = True
    assert torch.equal(torch.isnan(qo).any(-1), bad)


def test_empty(ops):
    q, f = rand(1, 0, 4, 128), freqs((64,))
    qo, ko = ops.qk_norm_rope(q, rand(1, 0, 2, 128), torch.zeros(0, dtype=torch.int64, device="cuda"), f)
    assert qo.shape == q.shape and ko.shape == (0, 2, 128)


def test_keys_need_queries(ops):
    pos, f = torch.arange(6, device="cuda"), freqs((64,))
    with pytest.raises(RuntimeError, match="q has no heads"):
        ops.qk_norm_rope(rand(1, 6, 0, 128), rand(2, 6, 2, 128), pos, f)
    qo, ko = ops.qk_norm_rope(rand(1, 6, 4, 128), rand(2, 6, 0, 128), pos, f)
    assert qo.shape == (6, 4, 128) and ko.shape == (6, 0, 128)


def test_given_outputs_count_as_changed(ops):
    q, k, pos, f = rand(1, 6, 4, 128), rand(2, 6, 2, 128), torch.arange(6, device="cuda"), freqs((64,))
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    saved = [(q * w).sum(), (k * w).sum()]  # keep q and k for the gradient of w
    ops.qk_norm_rope(q, k, pos, f, out=(q, k))
    for y in saved:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_refusals(ops):
    q, k, pos, f = rand(1, 6, 4, 128), rand(2, 6, 2, 128), torch.arange(6, device="cuda"), freqs((64,))
    w = rand(3, 128)
    bad = [
        lambda: ops.qk_norm_rope(q.float(), k, pos, f),
        lambda: ops.qk_norm_rope(q, k[:5], pos, f),
        lambda: ops.qk_norm_rope(q, k[None], pos, f),
        lambda: ops.qk_norm_rope(q[..., :64], k, pos, f),
        lambda: ops.qk_norm_rope(q, k, pos[:5], f),
        lambda: ops.qk_norm_rope(q, k, pos.double(), f),
        lambda: ops.qk_norm_rope(q, k, pos.cpu(), f),
        lambda: ops.qk_norm_rope(q, k, pos, f.double()),
        lambda: ops.qk_norm_rope(q, k, pos, f[::2]),
        lambda: ops.qk_norm_rope(q, k, pos, f, q_weight=w[:64]),
        lambda: ops.qk_norm_rope(q, k, pos, f, q_weight=w, k_weight=w.float()),
        lambda: ops.qk_norm_rope(q, None, pos, f, k_weight=w),
        lambda: ops.qk_norm_rope(q.clone().requires_grad_(), k, pos, f),
        lambda: ops.qk_norm_rope(q, k, pos, f, eps=-1.0),
        lambda: ops.qk_norm_rope(q, k, pos, f, out=(torch.empty_like(q)[:5], torch.empty_like(k))),
        lambda: ops.qk_norm_rope(q[1:], k[1:], pos[1:], f, out=(q[:-1], torch.empty_like(k[1:]))),   # one row off
        lambda: ops.qk_norm_rope(q, k, pos, f, out=(q[:, :1].expand(6, 4, 128), torch.empty_like(k))),
        lambda: ops.qk_norm_rope(q, q, pos, f, out=(q, q)),
        lambda: ops.qk_norm_rope(torch.zeros(6 * 512 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(6, 4, 128), k, pos, f),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")
    for kw in (dict(sections=(32, 31)), dict(sections=(70,)), dict(sections=(16,) * 5), dict(sections=())):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(q, k, pos, f, **kw)
