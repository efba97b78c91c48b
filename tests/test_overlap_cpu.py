"""CPU tests of the rules on where an output may lie."""

import random

import pytest
import torch

from b200_attention_b200 import _native as N


def places(t):
    """Bytes of a tensor, each as often as an element covers it."""
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return (t.data_ptr() + t.element_size() * at.reshape(-1, 1) + torch.arange(t.element_size())).reshape(-1)


def share(a, b):
    return bool(torch.isin(places(a), places(b)).any())


def test_random_views_against_their_elements(native_built):
    """Views of one buffer with any sizes and strides: the answer is the one that their elements give."""
    rng, both = random.Random(3), [0, 0]
    buf = torch.zeros(6000, dtype=torch.bfloat16)
    for _ in range(4000):
        views = []
        for _ in range(2):
            run = rng.choice([1, 2, 4, 8])
            sizes = [rng.randint(1, 5) for _ in range(rng.randint(0, 3))]
            strides = [rng.choice([0, 1, 3, run, 2 * run, 3 * run, 5 * run, 16, 24, 48, 64, 100, 144]) for _ in sizes]
            views.append(buf.as_strided(sizes + [run], strides + [1], rng.randint(0, 400)))
        want = share(*views)
        assert N.direct().may_overlap(*views) == want and N.direct().may_overlap(*views[::-1]) == want
        both[want] += 1
    assert min(both) > 500


def test_layouts_that_calls_come_with(native_built):
    """Columns of fused rows, heads in front of tokens, samples in between, other element sizes."""
    may = N.direct().may_overlap
    rows = torch.zeros(3, 70, 12, 128, dtype=torch.bfloat16)
    q, k, v = rows[:, :, :8], rows[:, :, 8:10], rows[:, :, 10:]
    assert not may(q, k) and not may(k, v) and not may(q, v) and may(q, rows[:, :, 7:9]) and may(q, q)
    by_head = torch.zeros(3, 12, 70, 128, dtype=torch.bfloat16).transpose(1, 2)
    q, k = by_head[:, :, :8], by_head[:, :, 8:]
    assert not may(q, k) and may(q, by_head[:, :, 7:]) and not may(q[:, :30], q[:, 30:]) and may(q[:, :31], q[:, 30:])
    base = torch.zeros(1000, dtype=torch.int32)
    assert may(base[100:], base.view(torch.bfloat16)[200:300]) and not may(base[:100], base.view(torch.bfloat16)[200:300])
    assert not may(base[:0], base) and not may(base, base[5:5])
    # samples that lie in one another's rows: apart by their columns, not by their rows
    x = torch.zeros(4096, dtype=torch.bfloat16)
    a, b = x.as_strided((2, 2, 1, 128), (384, 256, 128, 1)), x[128:].as_strided((2, 2, 1, 128), (384, 256, 128, 1))
    assert share(a, b) and may(a, b)


@pytest.mark.parametrize("make, fits", [
    (lambda r: (torch.zeros(6, 4, 128), r[:, :4], r[:, 4:]), True),                # a tensor of its own
    (lambda r: (r[:, :4], r[:, :4], r[:, 4:]), True),                              # q itself
    (lambda r: (r[:, 4:], r[:, :4], torch.zeros(6, 4, 128)), True),                # beside q in the same rows
    (lambda r: (r[:5, :4], r[1:, :4], torch.zeros(5, 4, 128)), False),             # q, one row off
    (lambda r: (r[:, 1:5], r[:, :4], torch.zeros(6, 4, 128)), False),              # q, one head off
    (lambda r: (r[:, 4:], r[:, :4], r[:, 4:]), False),                             # k
    (lambda r: (r[:, :4], r[:, :4], r[:, 3:]), False),                             # q, which k shares heads with
    (lambda r: (r[:, :1].expand(6, 4, 128), torch.zeros(6, 4, 128), torch.zeros(6, 4, 128)), False),   # heads on one another
    (lambda r: (r.as_strided((6, 4, 128), (128, 128, 1)), torch.zeros(6, 4, 128), torch.zeros(6, 4, 128)), False),
])
def test_where_a_result_may_lie(native_built, make, fits):
    out, q, k = make(torch.zeros(6, 8, 128))
    if fits:
        N.direct().check_place(out, q, k)
    else:
        with pytest.raises(RuntimeError, match="overlaps|share memory"):
            N.direct().check_place(out, q, k)
