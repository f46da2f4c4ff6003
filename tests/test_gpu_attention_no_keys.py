"""The C ABI's backward pass of attention without keys: dq is zeros, and there is nothing to write for dk and dv."""
import ctypes

import pytest
import torch

from nanotron_amd import _native as nt
from nanotron_amd import _ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CODES = {torch.bfloat16: nt.BF16, torch.float16: nt.F16}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rows", [500, 5000])
@pytest.mark.parametrize("wanted", ["qkv", "kv", "q", "v"])
def test_backward_without_keys(wanted, rows, packed, dtype):
    heads, kv_heads, dim = 8, 2, 64
    q, do = (torch.randn(rows, heads, dim, device=DEV).to(dtype) for _ in range(2))
    out, dq = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    dk, dv = (torch.full((64, kv_heads, dim), 7.0, device=DEV, dtype=dtype) for _ in range(2))   # (of no rows: left as they are)
    lse = torch.empty(heads, rows, device=DEV)
    cu = torch.tensor([0, rows], dtype=torch.int32, device=DEV), torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    d = _ops.AttentionDesc(q=q.data_ptr(), q_stride=heads * dim, q_head=dim, sequences=1, q_rows=rows, k_rows=0, heads=heads, kv_heads=kv_heads, head_dim=dim, dtype=CODES[dtype],
                           causal=1, scale=0.125, out=out.data_ptr(), lse=lse.data_ptr(), do_stride=heads * dim, do_head=dim)
    if packed:
        d.cu_q, d.cu_k = (t.data_ptr() for t in cu)
    room = torch.empty(max(_ops.lib.ntops_attention_workspace(ctypes.byref(d), b) for b in (0, 1)) + 256, dtype=torch.uint8, device=DEV)
    d.workspace = (room.data_ptr() + 255) // 256 * 256
    stream = torch.cuda.current_stream().cuda_stream
    assert _ops.lib.ntops_attention_forward(ctypes.byref(d), stream) == 0
    d.dout = do.data_ptr()
    d.dq, d.dk, d.dv = (t.data_ptr() if n in wanted else None for t, n in ((dq, "q"), (dk, "k"), (dv, "v")))
    assert _ops.lib.ntops_attention_backward(ctypes.byref(d), stream) == 0
    torch.cuda.synchronize()
    assert not out.any() and torch.isneginf(lse).all()
    assert not dq.any() if "q" in wanted else (dq == 7).all()
    assert (dk == 7).all() and (dv == 7).all()
