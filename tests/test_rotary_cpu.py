"""CPU tests of the norm-and-rotation entry point: refusals, before a device is touched."""

import ctypes as C

import pytest
import torch

from b200_attention_b200 import _native as N
from b200_attention_b200 import ops, rotary


def args(**over):
    a = N.QkNormRopeArgs()
    a.struct_bytes = C.sizeof(N.QkNormRopeArgs)
    a.batch, a.tokens, a.heads_q, a.heads_k, a.head_dim = 1, 4, 4, 2, 128
    a.q = a.q_out = N.Operand(0x10000, 0, 128, 512)
    a.k = a.k_out = N.Operand(0x20000, 0, 128, 256)
    a.positions = a.inv_freq = 0x30000
    a.axes, a.eps = 1, 1e-6
    a.section[0] = 64
    for key, val in over.items():
        if key == "section":
            a.section[:] = val
        else:
            setattr(a, key, val)
    return a


@pytest.mark.parametrize("over, status", [
    (dict(struct_bytes=8), N.STATUS_INVALID_ARGUMENT),
    (dict(reserved=1), N.STATUS_INVALID_ARGUMENT),
    (dict(head_dim=64), N.STATUS_UNSUPPORTED),
    (dict(tokens=0), N.STATUS_INVALID_ARGUMENT),
    (dict(heads_q=0), N.STATUS_INVALID_ARGUMENT),
    (dict(heads_k=-1), N.STATUS_INVALID_ARGUMENT),
    (dict(heads_q=65535), N.STATUS_UNSUPPORTED),
    (dict(batch=2**16, tokens=2**16), N.STATUS_UNSUPPORTED),
    (dict(axes=0), N.STATUS_INVALID_ARGUMENT),
    (dict(axes=5), N.STATUS_INVALID_ARGUMENT),
    (dict(section=[65, 0, 0, 0]), N.STATUS_INVALID_ARGUMENT),
    (dict(section=[0, 0, 0, 0]), N.STATUS_INVALID_ARGUMENT),
    (dict(axes=2, section=[40, 25, 0, 0]), N.STATUS_INVALID_ARGUMENT),
    (dict(axes=2, section=[40, -1, 0, 0]), N.STATUS_INVALID_ARGUMENT),
    (dict(weight_type=2), N.STATUS_INVALID_ARGUMENT),
    (dict(position_type=3), N.STATUS_INVALID_ARGUMENT),
    (dict(positions=0), N.STATUS_INVALID_ARGUMENT),
    (dict(inv_freq=0), N.STATUS_INVALID_ARGUMENT),
    (dict(eps=-1.0), N.STATUS_INVALID_ARGUMENT),
    (dict(eps=float("nan")), N.STATUS_INVALID_ARGUMENT),
    (dict(q=N.Operand(0, 0, 128, 512)), N.STATUS_INVALID_ARGUMENT),
    (dict(q_out=N.Operand(0x10008, 0, 128, 512)), N.STATUS_INVALID_ARGUMENT),
    (dict(k=N.Operand(0x10000, 0, 128, 257)), N.STATUS_INVALID_ARGUMENT),
    (dict(k_out=N.Operand(0, 0, 128, 256)), N.STATUS_INVALID_ARGUMENT),
])
def test_refused_before_touching_a_device(native_built, over, status):
    assert N.lib().b200attn_qk_norm_rope(C.byref(args(**over))) == status
    assert N.lib().b200attn_last_error() != b""


def test_null(native_built):
    assert N.lib().b200attn_qk_norm_rope(None) == N.STATUS_INVALID_ARGUMENT


def test_cpu_tensors_are_refused():
    x, f = torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.qk_norm_rope(x, x, torch.arange(4), f)
    with pytest.raises(TypeError):
        ops.qk_norm_rope([1.0], x, torch.arange(4), f)


def test_overlap_rule():
    """Which pairs of output and input may share memory: apart, or heads side by side in the same rows."""
    rows = torch.zeros(2, 5, 8, 128, dtype=torch.bfloat16)
    q, k, v = rows[:, :, :4], rows[:, :, 4:6], rows[:, :, 6:]
    for a, b in [(q, k), (k, v), (q, v), (q[:1], q[1:]), (q, torch.zeros_like(q))]:
        assert not rotary._may_overlap(a, b) and not rotary._may_overlap(b, a)
    assert rotary._may_overlap(q, rows[:, :, 3:7]) and rotary._may_overlap(q, q)
    assert rotary._may_overlap(rows[0, :4, :4], rows[0, 1:, :4])  # the same rows, one further
    assert rotary._same_place(q, rows[:, :, :4]) and not rotary._same_place(q, k)
    assert rotary._dense_apart(q) and not rotary._dense_apart(rows[:, :1].expand(2, 5, 8, 128))
