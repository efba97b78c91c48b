"""A bounded device-side wait of the planned attention kernel that runs out, and a table that is none.

As in test_gpu_wait_limit.py: a variant of the library is compiled in which one softmax warp withholds one barrier arrival
(on the second K/V tile of a CTA's first piece); the kernel gives up after 20 ms, says where, and the device stays usable.
Nothing traps, faults or spins without a limit."""

import ctypes as C

import pytest
import torch

from tests import packed_reference as R
from tests.test_gpu_wait_limit import _build_variant

pytestmark = pytest.mark.gpu

SITES = {110, 111, 114, 115, *range(100, 108),                 # TMA warp
         200, 201, 202, 203, 204, 210, 211, 212, 220, 221, 240, 241,  # MMA warp
         300, 301, 310, 311, 410, 411, 420, 421, 430, 431, 600}       # softmax, epilogue, V tails


def args_for(N, q, k, v, o, schedule, table):
    a = N.PlannedArgs()
    a.struct_bytes = C.sizeof(N.PlannedArgs)
    a.heads, a.heads_kv, a.head_dim = q.shape[1], k.shape[1], 128
    a.rows_q, a.rows_kv = q.shape[0], k.shape[0]
    a.grid, a.join_units, a.slot_rows = schedule.info.grid, schedule.info.units, schedule.info.slot_rows
    a.wide_pieces = schedule.info.wide_pieces
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, name, N.Operand(t.data_ptr(), 0, t.stride(1), t.stride(0)))
    a.table = table.data_ptr()
    a.stream = torch.cuda.current_stream().cuda_stream
    assert schedule.info.slot_rows == 0 and schedule.info.units == 0  # no workspace needed here
    return a


def rand(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def test_a_wait_that_runs_out_is_reported_and_the_device_stays_usable(native_built, tmp_path):
    from b200_attention_b200 import _native as N
    from b200_attention_b200.packed import Schedule

    lib = C.CDLL(str(_build_variant(tmp_path)))
    lib.b200attn_forward_planned.argtypes = [C.POINTER(N.PlannedArgs)]
    lib.b200attn_device_check.argtypes = [C.c_int, C.POINTER(C.c_int32)]
    lib.b200attn_set_wait_limit_ms.argtypes = [C.c_uint32]
    assert lib.b200attn_set_wait_limit_ms(20) == 0
    rec = (C.c_int32 * 8)()
    for lens_q, lens_kv, fails in [([200], [330], True), ([1, 1], [200, 150], True), ([1, 30], [100, 100], False)]:
        # pieces of two Q tiles; two lanes; pieces of one K/V tile, which never reach the withheld arrival
        q, k, v = rand(1, sum(lens_q), 2, 128), rand(2, sum(lens_kv), 2, 128), rand(3, sum(lens_kv), 2, 128)
        s = Schedule(lens_q, lens_kv, heads=2, sm_count=1)  # one CTA: nothing is cut
        table, o = s.table.cuda(), torch.empty_like(q)
        assert lib.b200attn_forward_planned(C.byref(args_for(N, q, k, v, o, s, table))) == 0
        torch.cuda.synchronize()  # the kernel ends by itself
        if fails:
            assert lib.b200attn_device_check(-1, rec) == N.STATUS_DEVICE_TIMEOUT
            assert rec[0] == 1 and rec[1] in SITES and rec[2] == 0 and 0 <= rec[3] < 16
        assert lib.b200attn_device_check(-1, rec) == N.STATUS_OK
        if not fails:
            R.check_attention(o, None, R.attention(q, k, v, lens_q, lens_kv, causal=True))


def test_a_table_that_is_none_is_refused_by_the_kernel(native_built):
    """What a captured call would find whose plan's memory had been given to somebody else: zeros here."""
    from b200_attention_b200 import _native as N
    from b200_attention_b200.packed import Schedule

    q, k, v = rand(1, 5, 2, 128), rand(2, 5, 2, 128), rand(3, 5, 2, 128)
    s = Schedule([5], [5], heads=2)
    o = torch.full_like(q, 2.0)
    none = torch.zeros_like(s.table).cuda()
    a = args_for(N, q, k, v, o, s, none)
    a.join_units = 8
    N.check(N.lib().b200attn_forward_planned(C.byref(a)))
    torch.cuda.synchronize()
    with pytest.raises(N.B200AttnError) as info:
        N.device_check()
    assert info.value.status == N.STATUS_DEVICE_FAULT
    assert (o == 2).all()
    N.device_check()
