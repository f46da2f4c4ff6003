"""Sizes at which a product of two arguments leaves 32 or 64 bits: the C ABI of the operators of a decoder layer refuses them before any launch."""
import pytest
from test_layer_ops_capi import ALIAS, SIZE, attend, turns

from nanotron_amd import _ops


@pytest.mark.parametrize("kw", [dict(pairs=1 << 30), dict(pairs=(1 << 31) - 1), dict(pairs=(1 << 30) + 16), dict(heads=(1 << 31) - 1, kv_heads=(1 << 31) - 1),
                                dict(tokens=(1 << 31) - 1, q_stride=1 << 31), dict(tokens=(1 << 31) - 1, k_stride=1 << 31)])
def test_rotary_sizes_beyond_their_products(kw):
    assert _ops.lib.ntops_rotary(turns(**kw), None) == SIZE


@pytest.mark.parametrize("count", [4, 1 << 58, (1 << 62) + 4])
def test_rotary_positions_over_an_output(count):
    """The third of the four positions that are read is where the rotated queries go, however many more there are said to be."""
    assert _ops.lib.ntops_rotary(turns(positions=0x300000 - 0x10, position_count=count), None) == ALIAS


@pytest.mark.parametrize("kw", [dict(heads=1 << 20, kv_heads=1, k_stride=64, q_head=1 << 45), dict(heads=1 << 20, kv_heads=1 << 20, k_head=1 << 45), dict(heads=1 << 20, kv_heads=1 << 20, v_head=1 << 46),
                                dict(sequences=1 << 20, q_rows=1 << 20, k_rows=1 << 20, heads=1, kv_heads=1, q_batch=1 << 45),
                                dict(sequences=1 << 20, q_rows=1 << 20, k_rows=1 << 20, heads=1, kv_heads=1, v_batch=1 << 45)])
def test_attention_distances_beyond_64_bits(kw):
    assert _ops.lib.ntops_attention_forward(attend(**kw), None) == SIZE


@pytest.mark.parametrize("kw", [dict(heads=1 << 20, kv_heads=1 << 20, do_head=1 << 45), dict(sequences=1 << 20, q_rows=1 << 20, k_rows=1 << 20, heads=1, kv_heads=1, do_batch=1 << 45)])
def test_attention_gradients_distances_beyond_64_bits(kw):
    grad = dict(dout=0x60000000, lse=0x70000000, dq=0x80000000, dk=0x90000000, dv=0xa0000000)
    assert _ops.lib.ntops_attention_backward(attend(**grad, **kw), None) == SIZE


def test_distances_that_nothing_uses_are_not_looked_at():
    """Sequences that are packed have no distance from one to the next, a forward call no gradient: what stands there then leads no further than a refusal for another reason."""
    packed = dict(cu_q=0x6000000, cu_k=0x6000000, sequences=1 << 18)
    for kw in (dict(q_batch=1 << 45, k_batch=1 << 45, do_batch=1 << 45, **packed), dict(heads=1 << 10, kv_heads=1 << 10, do_head=1 << 45)):
        assert _ops.lib.ntops_attention_forward(attend(out=0x1000100, **kw), None) == ALIAS
