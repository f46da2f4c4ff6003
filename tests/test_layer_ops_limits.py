"""Sizes at which a product of two arguments leaves 32 or 64 bits: the C ABI of the operators of a decoder layer refuses them before any launch."""
import pytest
from test_layer_ops_capi import ALIAS, SIZE, turns

from nanotron_amd import _ops


@pytest.mark.parametrize("kw", [dict(pairs=1 << 30), dict(pairs=(1 << 31) - 1), dict(pairs=(1 << 30) + 16), dict(heads=(1 << 31) - 1, kv_heads=(1 << 31) - 1),
                                dict(tokens=(1 << 31) - 1, q_stride=1 << 31), dict(tokens=(1 << 31) - 1, k_stride=1 << 31)])
def test_rotary_sizes_beyond_their_products(kw):
    assert _ops.lib.ntops_rotary(turns(**kw), None) == SIZE


@pytest.mark.parametrize("count", [4, 1 << 58, (1 << 62) + 4])
def test_rotary_positions_over_an_output(count):
    """The third of the four positions that are read is where the rotated queries go, however many more there are said to be."""
    assert _ops.lib.ntops_rotary(turns(positions=0x300000 - 0x10, position_count=count), None) == ALIAS
