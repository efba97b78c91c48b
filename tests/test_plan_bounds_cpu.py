"""CPU tests: no piece of a schedule is longer than a CTA may walk without a look at the others."""

import random

import pytest

from b200_attention_b200 import packed

PIECE_AT = 2576      # words of the table in front of the pieces
LONGEST = 1 << 15    # K/V tiles of a piece: under a tenth of a second, well inside the limit of the device-side waits


def longest_piece(lens_q, lens_kv, **kw):
    s = packed.Schedule(lens_q, lens_kv, **kw)
    pieces = s.table.numpy()[PIECE_AT:PIECE_AT + 12 * s.info.pieces].reshape(-1, 12)
    return int(pieces[:, 4:6].max())


@pytest.mark.parametrize("lens_q, lens_kv, heads, heads_kv, sm_count", [
    ([1392, 1237], [52625857, 64133829], 8, 2, 148),
    ([1] * 4, [21_000_000, 26_000_000, 30_000_000, 35_000_000], 1, 1, 8),
    ([300] * 4, [21_000_000, 26_000_000, 30_000_000, 35_000_000], 2, 2, 8),
    ([1], [2**30 - 1], 1, 1, 1),
    ([1], [(LONGEST + 1) * 128], 8, 8, 148),
])
def test_pieces_of_very_long_rows_are_bounded(native_built, lens_q, lens_kv, heads, heads_kv, sm_count):
    """Sequences that share their keys, so that such lengths fit a device's memory."""
    got = longest_piece(lens_q, lens_kv, heads=heads, heads_kv=heads_kv, sm_count=sm_count, causal=False,
                        starts_kv=[0] * len(lens_kv))
    assert got <= LONGEST


def test_pieces_on_a_very_long_prefix_are_bounded(native_built):
    assert longest_piece([3, 4], [3, 4], heads=8, heads_kv=2, sm_count=4, len_prefix=60_000_000) <= LONGEST


def test_random_very_long_rows_are_bounded(native_built):
    rng = random.Random(7)
    for _ in range(300):
        n = rng.randint(1, 5)
        lens_q = [rng.choice([1, rng.randint(1, 1500)]) for _ in range(n)]
        lens_kv = [rng.randint(1_000_000, 80_000_000) for _ in range(n)]
        heads_kv = rng.choice([1, 2, 8])
        got = longest_piece(lens_q, lens_kv, heads=heads_kv * rng.choice([1, 4]), heads_kv=heads_kv,
                            sm_count=rng.choice([4, 16, 148]), causal=False, starts_kv=[0] * n)
        assert got <= LONGEST
