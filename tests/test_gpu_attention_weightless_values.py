"""A value that is not finite reaches every row of attention that sees its key, however small that key's share."""
import math

import pytest
import torch
from test_gpu_attention import DEV, exact, near

from nanotron_amd.nn import attention

pytestmark = pytest.mark.gpu
E = 5   # the element of a head that tells keys apart


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("tokens, keys", [(1, 40), (1, 500), (4, 200), (1, 2000), (100, 3000), (200, 200)])
def test_a_value_of_no_weight_that_is_not_finite_arrives(tokens, keys, bad):
    """The first half of the keys (32 at least) scores 180 (base 2) below the others, so that their share is 0 in fp32: what is infinite among their values makes the element of the output
    infinite in exact arithmetic, and 0 times infinity in this."""
    heads, kv_heads, dim = 4, 2, 64
    g = torch.Generator().manual_seed(keys)
    q = torch.randn(1, tokens, heads, dim, generator=g).bfloat16().to(DEV)
    k, v = (torch.randn(1, keys, kv_heads, dim, generator=g).bfloat16().to(DEV) for _ in range(2))
    q[..., E], k[..., E] = 32.0, 0.0
    k[:, :max(32, keys // 2), :, E] = -32.0
    args = [t.flatten(0, 1) for t in (q, k, v)]
    want, bound = exact(*args, torch.zeros_like(args[0]), [(tokens, keys)], causal=False)
    v[0, 3, 1, 7] = bad
    with torch.no_grad():
        out = attention(q, k, v, causal=False).flatten(0, 1)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[:, 2:, 7] = True
    assert torch.equal(~torch.isfinite(out), hit)
    near(out[~hit], want[0][~hit], bound[0][~hit], "out")
