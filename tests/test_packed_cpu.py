"""CPU tests of the planned attention calls: the schedule covers every (token, key) pair exactly once and joins what it
cuts, and everything that a call or a plan refuses is refused before a device is touched."""

import ctypes as C
import random

import numpy as np
import pytest
import torch

from b200_attention_b200 import _native as N
from b200_attention_b200 import ops, packed

CTA_AT, PIECE_AT = 16, 2576  # words: a record for each CTA (bounds of its pieces and a copy of the first), pieces


def expand(lens_q, lens_kv, heads, heads_kv, *, causal, starts=None, prefix=0, sm_count=0):
    """Checks a schedule's table by walking it, row by row; returns it."""
    s = packed.Schedule(lens_q, lens_kv, heads=heads, heads_kv=heads_kv, causal=causal, starts_kv=starts,
                        len_prefix=prefix, sm_count=sm_count)
    t, info = s.table.numpy(), s.info
    group = heads // heads_kv
    per_tile = 128 // group
    records = t[CTA_AT:PIECE_AT].reshape(160, 16)
    ctas = records[:, :4]  # pieces of two Q tiles, lane 0's, lane 1's, end
    assert ctas[0, 0] == 0 and ctas[-1, 3] == info.pieces == t[1] and (np.diff(ctas.ravel()) >= 0).all()
    assert (ctas[1:, 0] == ctas[:-1, 3]).all()
    assert (ctas[info.grid:, 0] == info.pieces).all() and info.grid <= (sm_count or 148)
    assert info.workspace_bytes == info.slot_rows * 129 * 4 and info.table_bytes == 4 * t.size
    pieces = t[PIECE_AT:PIECE_AT + 12 * info.pieces].reshape(-1, 12)
    units = t[t[3]:t[3] + 8 * info.units].reshape(-1, 8)
    parts = t[t[4]:]
    for record in records[ctas[:, 0] < ctas[:, 3]]:
        assert (record[4:] == pieces[record[0]]).all()
    both = pieces[:, 5] > 0
    for pairs, lane0, lane1, end in ctas.tolist():
        assert both[pairs:lane0].all() and not both[lane0:end].any()
        assert lane1 > lane0 or end == lane1, "lane 1 has work, lane 0 none"
        for a, b in ((lane0, lane1), (lane1, end)):  # pieces that fill the lane's Q buffer come before those that share it
            small = pieces[a:b, 1] <= 32 // group
            assert (small[:-1] <= small[1:]).all()
    runs, slot_owner = {}, {}
    for token, n, row, keys, tiles0, tiles1, diag, head, source, slot in pieces[:, :10].tolist():
        assert 1 <= n <= 2 * per_tile and keys > 0 and tiles0 >= 1
        assert (tiles1 >= tiles0) if n > per_tile else tiles1 == 0
        for j in range(n):
            tiles = tiles0 if j < per_tile else tiles1
            seen = max(0, min(keys, diag + j + 1, 128 * tiles))
            runs.setdefault((token + j, head), []).append((source, row, row + seen, slot))
            for g in range(group if slot >= 0 else 0):
                at = slot + j * group + g
                assert at not in slot_owner and at < info.slot_rows
                slot_owner[at] = (token + j, head, g)
    joined = {}
    for token, n, head, part0, count in units[:, :5].tolist():
        assert n >= 1 and (n == 1 or n * group <= 32)
        for j in range(n):
            assert (token + j, head) not in joined
            joined[token + j, head] = count
            for part in parts[part0:part0 + count].tolist():
                for g in range(group):
                    assert slot_owner.pop(part + j * group + g) == (token + j, head, g)
    assert not slot_owner, "partial rows that nobody joins"
    first = np.concatenate([[0], np.cumsum(lens_kv)]).tolist() if starts is None else starts
    token = 0
    for n, m, start in zip(lens_q, lens_kv, first):
        for j in range(n):
            for head in range(heads_kv):
                mine = runs.pop((token, head), [])
                own = sorted(r[1:3] for r in mine if r[0] == 0 and r[2] > r[1])
                want = max(0, min(m, m - n + j + 1)) if causal else m
                at = start
                for a, b in own:
                    assert a == at
                    at = b
                assert at == start + want
                at = 0
                for a, b in sorted(r[1:3] for r in mine if r[0] == 1):
                    assert a == at
                    at = b
                assert at == prefix
                if (token, head) in joined:
                    assert joined[token, head] == len(mine) and all(r[3] >= 0 for r in mine)
                else:
                    assert len(mine) == 1 and mine[0][3] == -1
            token += 1
    assert not runs and info.rows_q == token
    assert info.rows_kv == max([a + m for a, m in zip(first, lens_kv) if m], default=0)
    return s


@pytest.mark.parametrize("lens_q, lens_kv, heads, heads_kv, causal, prefix", [
    ([1], [1], 1, 1, True, 0),
    ([0], [5], 2, 1, True, 0),                        # nothing to do
    ([3], [0], 4, 2, False, 0),                       # no key: joined from nothing
    ([200, 1, 129], [5, 1, 129], 4, 4, True, 0),      # rows that see nothing, whole tiles of them
    ([1], [30000], 8, 1, True, 0),                    # one token, cut into many pieces
    ([1] * 40, [1000 + 37 * i for i in range(40)], 16, 2, True, 0),
    ([600], [600], 3, 1, True, 0),                    # 42 tokens to a tile
    ([70], [700], 128, 1, True, 0),                   # one token to a tile
    ([2, 1, 3], [2, 9, 300], 8, 2, True, 5000),       # prefix
    ([300, 0, 1], [300, 0, 1], 10, 2, True, 129),     # prefix blocks across sequences
    ([1, 1], [0, 0], 2, 2, False, 77),                # prefix alone
])
def test_schedule_covers_every_pair_once(native_built, lens_q, lens_kv, heads, heads_kv, causal, prefix):
    expand(lens_q, lens_kv, heads, heads_kv, causal=causal, prefix=prefix)


def test_random_schedules(native_built):
    rng = random.Random(11)
    done = cut = 0
    while done < 150:
        heads_kv, group = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 3, 4, 5, 8, 16])
        count, top = rng.randint(1, 6), rng.choice([3, 40, 300, 1500])
        lens_q = [rng.choice([0, 1, rng.randint(0, top)]) for _ in range(count)]
        if sum(lens_q) * heads_kv > 3000:
            continue
        causal, prefix = rng.random() < 0.6, rng.choice([0, 0, 1, 128, 1000, 5000])
        lens_kv = [rng.choice([0, n, n + rng.randint(0, 4000), rng.randint(0, top)]) for n in lens_q]
        if prefix and causal:
            lens_kv = [max(a, b) for a, b in zip(lens_q, lens_kv)]
        starts = [rng.randint(0, 10**6) for _ in lens_kv] if rng.random() < 0.4 else None
        s = expand(lens_q, lens_kv, heads_kv * group, heads_kv, causal=causal, starts=starts, prefix=prefix,
                   sm_count=rng.choice([0, 0, 160, 16, 1]))
        done += 1
        cut += s.info.slot_rows > 0
    assert cut > 30


def test_work_is_spread_evenly(native_built):
    """Pieces go to the CTA that is free first, so when a CTA took its last one no other had less: its load is at most
    the mean load and one piece more. Counted in K/V tiles; a piece's start counts as up to 2."""
    for lens_q, lens_kv, heads, heads_kv in [([16384], [16384], 16, 16), ([1], [65536], 32, 8),
                                             ([1] * 64, [100 + (i * 4463) % 11901 for i in range(64)], 32, 8),
                                             ([2500] * 5, [2500] * 5, 8, 2)]:
        s = packed.Schedule(lens_q, lens_kv, heads=heads, heads_kv=heads_kv)
        t = s.table.numpy()
        pieces = t[PIECE_AT:PIECE_AT + 12 * s.info.pieces].reshape(-1, 12)
        ctas = t[CTA_AT:PIECE_AT].reshape(160, 16)
        tiles = pieces[:, 4:6].max(1)
        load = [tiles[a:b].sum() for a, b in ctas[:148, [0, 3]]]
        assert max(load) <= np.mean(load) + 2 * s.info.pieces / 148 + tiles.max() + 2
    one = packed.Schedule([1], [65536], heads=32, heads_kv=8)
    assert one.info.grid == 148  # a single token's keys are cut so that every CTA has some


@pytest.mark.parametrize("kw, error", [
    (dict(lens_q=[], lens_kv=[]), N.B200AttnError),
    (dict(lens_q=[1, 2]), ValueError),
    (dict(lens_q=[-1]), ValueError),
    (dict(lens_kv=[2**30]), ValueError),
    (dict(lens_q=[1.5]), TypeError),
    (dict(lens_q=[True]), TypeError),
    (dict(lens_q=torch.tensor([1.0])), TypeError),
    (dict(starts_kv=[0, 1]), ValueError),
    (dict(starts_kv=[-1]), ValueError),
    (dict(starts_kv=[2**31 - 260]), N.B200AttnError),  # last key past the rows that a coordinate can name
    (dict(heads=0), N.B200AttnError),
    (dict(heads=4, heads_kv=3), N.B200AttnError),
    (dict(heads=4, heads_kv=0), N.B200AttnError),
    (dict(heads=129, heads_kv=1), N.B200AttnError),
    (dict(len_prefix=-1), N.B200AttnError),
    (dict(len_prefix=2**31), ValueError),
    (dict(lens_q=[9], lens_kv=[3], len_prefix=5), N.B200AttnError),  # causal, fewer own keys than queries
    (dict(sm_count=161), N.B200AttnError),
])
def test_plans_refused(native_built, kw, error):
    args = dict(lens_q=[4], lens_kv=[4], heads=4, heads_kv=2)
    args.update(kw)
    lens_q, lens_kv = args.pop("lens_q"), args.pop("lens_kv")
    with pytest.raises(error):
        packed.Schedule(lens_q, lens_kv, **args)


@pytest.mark.parametrize("kw", [dict(heads=2.5), dict(heads=4, heads_kv=2.0), dict(heads=4, len_prefix=1.5), dict(heads="4")])
def test_plans_take_integers_only(native_built, kw):
    with pytest.raises(TypeError):
        packed.Schedule([4], [4], **kw)


def test_plan_needs_a_cuda_device(native_built):
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.AttentionPlan([1], [1], heads=1, device="cpu")


def test_plan_entry_points_check_their_structures(native_built):
    lib = N.lib()
    d, info, handle = N.PlanDesc(), N.PlanInfo(), C.c_void_p()
    assert lib.b200attn_plan_create(None, C.byref(info), C.byref(handle)) == N.STATUS_INVALID_ARGUMENT
    assert lib.b200attn_plan_create(C.byref(d), C.byref(info), C.byref(handle)) == N.STATUS_INVALID_ARGUMENT
    d.struct_bytes, info.struct_bytes = C.sizeof(d), C.sizeof(info)
    assert lib.b200attn_plan_create(C.byref(d), C.byref(info), C.byref(handle)) == N.STATUS_INVALID_ARGUMENT  # no lengths
    d.sequences, d.heads, d.heads_kv = 1, 1, 1
    d.len_q = d.len_kv = (C.c_int32 * 1)(1)
    assert lib.b200attn_plan_create(C.byref(d), C.byref(info), C.byref(handle)) == N.STATUS_OK
    small = (C.c_int32 * 4)()
    assert lib.b200attn_plan_table(handle, small, 16) == N.STATUS_INVALID_ARGUMENT
    assert lib.b200attn_plan_table(None, small, 16) == N.STATUS_INVALID_ARGUMENT
    assert lib.b200attn_plan_destroy(handle) == N.STATUS_OK
    assert lib.b200attn_plan_destroy(None) == N.STATUS_OK


def planned_args(**over):
    a = N.PlannedArgs()
    a.struct_bytes = C.sizeof(N.PlannedArgs)
    a.heads, a.heads_kv, a.head_dim, a.rows_q, a.rows_kv, a.grid = 4, 2, 128, 8, 8, 1
    a.q = a.o = N.Operand(0x10000, 0, 128, 512)
    a.k = a.v = a.k_prefix = a.v_prefix = N.Operand(0x10000, 0, 128, 256)
    a.table = 0x10000
    for key, val in over.items():
        setattr(a, key, val)
    return a


@pytest.mark.parametrize("over, status", [
    (dict(struct_bytes=8), N.STATUS_INVALID_ARGUMENT),
    (dict(reserved=1), N.STATUS_INVALID_ARGUMENT),
    (dict(head_dim=64), N.STATUS_UNSUPPORTED),
    (dict(heads=3), N.STATUS_INVALID_ARGUMENT),
    (dict(heads=512, heads_kv=2), N.STATUS_UNSUPPORTED),
    (dict(rows_q=0), N.STATUS_INVALID_ARGUMENT),
    (dict(rows_kv=-1), N.STATUS_INVALID_ARGUMENT),
    (dict(rows_kv=0), N.STATUS_INVALID_ARGUMENT),                            # work, but no keys
    (dict(grid=161), N.STATUS_INVALID_ARGUMENT),
    (dict(join_units=-1), N.STATUS_INVALID_ARGUMENT),
    (dict(table=0), N.STATUS_INVALID_ARGUMENT),
    (dict(table=0x10008), N.STATUS_INVALID_ARGUMENT),
    (dict(slot_rows=4), N.STATUS_INVALID_ARGUMENT),                          # no workspace
    (dict(slot_rows=4, workspace=0x10010), N.STATUS_INVALID_ARGUMENT),
    (dict(lse=0x10000, lse_stride_head=7), N.STATUS_INVALID_ARGUMENT),
    (dict(softmax_scale=float("inf")), N.STATUS_INVALID_ARGUMENT),
    (dict(q=N.Operand(0, 0, 128, 512)), N.STATUS_INVALID_ARGUMENT),
    (dict(k=N.Operand(0x10008, 0, 128, 256)), N.STATUS_INVALID_ARGUMENT),
    (dict(v=N.Operand(0x10000, 0, 128, 260)), N.STATUS_INVALID_ARGUMENT),
    (dict(o=N.Operand(0x10000, 0, 64, 512)), N.STATUS_INVALID_ARGUMENT),
    (dict(len_prefix=5, k_prefix=N.Operand(0, 0, 128, 256)), N.STATUS_INVALID_ARGUMENT),
])
def test_planned_call_refuses_before_touching_a_device(native_built, over, status):
    assert N.lib().b200attn_forward_planned(C.byref(planned_args(**over))) == status
    assert N.lib().b200attn_last_error() != b""


def test_planned_call_null(native_built):
    assert N.lib().b200attn_forward_planned(None) == N.STATUS_INVALID_ARGUMENT


def test_calls_need_a_plan():
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="AttentionPlan"):
        ops.attention_packed(x, x, x, None)
    with pytest.raises(TypeError, match="AttentionPlan"):
        ops.attention_shared_prefix(x, x, x, x, x, [4])
