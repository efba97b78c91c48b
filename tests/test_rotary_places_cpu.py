"""CPU tests: which places of an output qk_norm_rope takes for apart from its inputs."""

import torch

from b200_attention_b200 import rotary


def test_heads_in_front_of_tokens_in_a_batch(native_built):
    """q and k of one buffer [batch, heads, tokens, 128]: every sample's q lies between two samples' k."""
    buf = torch.zeros(3, 6, 50, 128, dtype=torch.bfloat16).transpose(1, 2)
    q, k = buf[:, :, :4], buf[:, :, 4:]
    assert not rotary._may_overlap(q, k) and not rotary._may_overlap(k, q)
    assert rotary._may_overlap(q, buf[:, :, 3:])


def test_samples_that_lie_in_one_another(native_built):
    """Two samples, the second one token and a half further: its columns are those of the first one's next token."""
    x = torch.zeros(4096, dtype=torch.bfloat16)
    a, b = (x[at:].as_strided((2, 2, 1, 128), (384, 256, 128, 1)) for at in (0, 128))
    assert a[1, 0].data_ptr() == b[0, 1].data_ptr()
    assert rotary._may_overlap(a, b) and rotary._may_overlap(b, a)


def test_nothing_overlaps_an_empty_tensor(native_built):
    x = torch.zeros(4, 5, 8, 128, dtype=torch.bfloat16)
    assert not rotary._may_overlap(x, x[:, :0]) and not rotary._may_overlap(x[:, :, :0], x)
