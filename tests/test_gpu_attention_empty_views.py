"""Attention over the first zero positions of a cache, whatever the distances of a tensor without elements are."""
import pytest
import torch

from nanotron_amd.nn import attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("shape, dim", [((2, 10, 2, 100), 80), ((2, 10, 2, 67), 64), ((2, 10, 3, 128), 128)])
@pytest.mark.parametrize("tokens", [1, 5, 200])
def test_no_keys_of_a_cache_with_odd_distances(tokens, shape, dim):
    cache = torch.randn(shape, device=DEV).bfloat16()
    q = torch.randn(2, tokens, 6, dim, device=DEV).bfloat16()
    for view in (cache[..., :dim][:, :0], cache[:, :0, :, :dim], cache.transpose(0, 1)[:0, :, :, :dim].transpose(0, 1)):
        with torch.no_grad():
            out = attention(q, view, view)
        assert out.shape == q.shape and not out.any()
        leaves = [q.clone().requires_grad_(True), view.detach().requires_grad_(True)]
        got = torch.autograd.grad(attention(leaves[0], leaves[1], leaves[1]).sum(), leaves)
        assert not got[0].any() and got[1].shape == view.shape
    # packed
    view = cache[0, :0, :, :dim]
    cu = torch.tensor([0, tokens], dtype=torch.int32, device=DEV)
    for kw in (dict(), dict(cu_seqlens=cu, cu_seqlens_k=torch.zeros_like(cu))):
        with torch.no_grad():
            assert not attention(q[0], view, view, **kw).any()
