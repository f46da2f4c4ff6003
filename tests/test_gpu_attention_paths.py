"""Ways through attention's kernels that few sizes take: packed keys cut into runs, heads of a group beside each other with cut keys or with a last workgroup that has heads
for some of its waves, a backward pass that makes its own plan, and the eight bits that the output's rounding leaves out."""
import ctypes
import math

import pytest
import torch
from test_gpu_attention import DEV, U, W, check, exact, inputs, near, offsets, step

from nanotron_amd import _native as nt
from nanotron_amd import _ops
from nanotron_amd.nn import attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 2, 128), (4, 4, 64), (5, 1, 80)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", [[(1, 3000), (20, 2500)], [(200, 2100), (0, 1500), (3, 4000)], [(1, 1500), (70, 1300), (40, 0), (2, 3000)]])
def test_packed_keys_in_runs(lengths, causal, heads, kv_heads, dim):
    """More than 1024 keys a sequence on average, few queries: runs of keys, joined; rows in front of and behind the sequences are zeros."""
    n, m = (sum(x[i] for x in lengths) for i in range(2))
    q, k, v, do = inputs(n, heads, kv_heads, dim, torch.bfloat16, keys=m, seed=n)
    cu = offsets(lengths), offsets(lengths, 1)
    want, bound = exact(q, k, v, do, lengths, causal)
    with torch.no_grad():
        out = attention(q, k, v, cu_seqlens=cu[0], cu_seqlens_k=cu[1], causal=causal)
        near(out, want[0], bound[0], "out")
        pad = torch.full((7, heads, dim), math.nan, dtype=q.dtype, device=DEV)
        more = attention(torch.cat([pad, q, pad]), k, v, cu_seqlens=cu[0] + 7, cu_seqlens_k=cu[1], causal=causal)
    assert torch.equal(more[7:n + 7], out) and not more[:7].any() and not more[n + 7:].any()
    got = step(q, k, v, do, cu_seqlens=cu[0], cu_seqlens_k=cu[1], causal=causal)
    for a, w, b, name in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        near(a, w, b, name)


@pytest.mark.parametrize("heads, kv_heads", [(8, 2), (6, 1), (5, 1)])
@pytest.mark.parametrize("tokens", [20, 30])
def test_heads_beside_each_other_over_keys_in_runs(tokens, heads, kv_heads):
    """A batch with more than 32 rows a group and fewer than 32 queries."""
    b, keys, dim = 2, 4096, 64
    g = torch.Generator().manual_seed(tokens)
    q = (1.5 * torch.randn(b * tokens, heads, dim, generator=g)).bfloat16().to(DEV)
    k, v = (torch.randn(b * keys, kv_heads, dim, generator=g).bfloat16().to(DEV) for _ in range(2))
    do = torch.randn(b * tokens, heads, dim, generator=g).mul_(0.1).bfloat16().to(DEV)
    want, bound = exact(q, k, v, do, [(tokens, keys)] * b)
    got = step(q.view(b, tokens, heads, dim), k.view(b, keys, kv_heads, dim), v.view(b, keys, kv_heads, dim), do.view(b, tokens, heads, dim))
    for a, w, e, name in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        near(a.flatten(0, 1), w, e, name)


@pytest.mark.parametrize("heads, kv_heads", [(5, 1), (6, 1), (7, 1), (10, 2), (2, 1), (3, 1)])
@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 64), (torch.float16, 128)])
def test_packed_steps_with_heads_beside_each_other(dtype, dim, heads, kv_heads):
    lengths = [20, 7, 0, 33, 1, 31, 64, 5]
    n = sum(lengths)
    q, k, v, do = inputs(n, heads, kv_heads, dim, dtype, seed=heads)
    check(q, k, v, do, [(x, x) for x in lengths], cu_seqlens=offsets(lengths))
    batch = [t[:n // 3 * 3].unflatten(0, (3, n // 3)) for t in (q, k, v, do)]
    got = step(*batch)
    want, bound = exact(*(t.flatten(0, 1) for t in batch), [(n // 3, n // 3)] * 3)
    for a, w, e, name in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        near(a.flatten(0, 1), w, e, name)


def native(q, k, v, do, cu, plan, low):
    """(out, dq, dk, dv) through the C ABI, with or without a plan and the bits behind out's."""
    lib, stream = _ops.lib, torch.cuda.current_stream().cuda_stream
    (n, heads, dim), (m, kv_heads, _) = q.shape, k.shape
    out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    d = _ops.AttentionDesc(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=heads * dim, k_stride=kv_heads * dim, v_stride=kv_heads * dim, q_head=dim, k_head=dim, v_head=dim,
                           cu_q=cu.data_ptr(), cu_k=cu.data_ptr(), sequences=cu.numel() - 1, q_rows=n, k_rows=m, heads=heads, kv_heads=kv_heads, head_dim=dim,
                           dtype=nt.BF16 if q.dtype == torch.bfloat16 else nt.F16, causal=1, scale=dim ** -0.5, out=out.data_ptr(), do_stride=heads * dim, do_head=dim)
    lse, bits = torch.empty(heads, n, device=DEV), torch.empty(n, heads, dim, dtype=torch.uint8, device=DEV)
    d.lse, d.out_low = lse.data_ptr(), bits.data_ptr() if low else None

    def room(size):
        t = torch.empty(size + 256, dtype=torch.uint8, device=DEV)
        return t, (t.data_ptr() + 255) // 256 * 256

    kept, at = room(lib.ntops_attention_plan(ctypes.byref(d)))
    d.plan = at if plan else None
    for backward, f in enumerate((lib.ntops_attention_forward, lib.ntops_attention_backward)):
        if backward:
            d.dout, d.dq, d.dk, d.dv = (t.data_ptr() for t in (do, dq, dk, dv))
        work, d.workspace = room(lib.ntops_attention_workspace(ctypes.byref(d), backward))
        assert f(ctypes.byref(d), stream) == 0
        torch.cuda.synchronize()
    return out, dq, dk, dv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths, heads, kv_heads", [([200, 0, 37, 300], 4, 2), ([9, 20, 1, 33], 8, 2), ([1200], 2, 1)])
def test_backward_that_makes_its_own_plan(lengths, heads, kv_heads, dtype):
    q, k, v, do = inputs(sum(lengths), heads, kv_heads, 64, dtype, seed=5)
    cu = offsets(lengths)
    want, bound = exact(q, k, v, do, [(x, x) for x in lengths])
    first = step(q, k, v, do, cu_seqlens=cu)
    for plan in (True, False):
        for low in (True, False):
            got = native(q, k, v, do, cu, plan, low)
            for a, w, e, name in zip(got, want, bound, ("out", "dq", "dk", "dv")):
                near(a, w, e, name)
            # the plan reaches no bit, and the bits behind out's none of out and dv
            same = got if low else (got[0], got[3])
            assert all(torch.equal(a, b) for a, b in zip(same, first if low else (first[0], first[3])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n, m", [(40, 3), (3, 7), (64, 5), (300, 11)])
def test_what_outs_rounding_leaves_out_reaches_the_gradients(n, m, dtype):
    """Keys that are all alike have the same share, 1 / m, whatever the query, and dq = 0: ds = (dp - delta) / m, dp the gradient times a value and delta their mean.
    Values that differ by little make every dp - delta small beside delta, so that an error of out's own rounding, u |dout||out| in delta, would be most of dq.

    Bounds.  A score is the same number for every key, so numerators are equal, 1 + x with |x| <= (|c s| + 16) W, and the sum m times that within m W: out is off by
    e = (2 m + 2 |c s| + 32) W of its values' magnitudes, and by 2^-7 u |out| where 8 more bits are kept (half of one of them, a whole one where a tie has no code), fp16's smallest
    step 2^-25 besides.  dp is off by 72 W, delta by 72 W and out's; p by e; ds by all that and by its rounding, u |ds|.  The keys' equal
    element times the sum of the m errors, (m + 8) W more for adding up, is what dq may be."""
    u, dim, heads = U[dtype], 64, 2
    g = torch.Generator().manual_seed(n + m)
    unit = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -10     # of values between 1 and 2
    q = torch.randn(n, heads, dim, generator=g).to(dtype).to(DEV)
    k = torch.randn(1, 1, dim, generator=g).to(dtype).to(DEV).expand(m, 1, dim)
    v = (1.5 + unit * torch.randint(-1, 2, (m, 1, dim), generator=g).double()).to(dtype).to(DEV)
    do = torch.randn(n, heads, dim, generator=g).to(dtype).to(DEV)
    _, dq, _, _ = step(q, k, v, do, causal=False)
    Q, K, V, G = (t.double() for t in (q, k, v, do))
    s = (Q @ K[0, 0]).abs() * dim ** -0.5 * 1.4427
    o = V[:, 0].mean(0)
    e = (2 * m + 2 * s[..., None] + 32) * W
    e_out = e * o.abs() + (2.0 ** -7 * u + 72 * W) * o.abs() + (2.0 ** -25 * 2.0 ** -7 if dtype == torch.float16 else 0.0)
    dp = G @ V[:, 0].t()                                            # [n, heads, m]
    delta = (G @ o)[..., None]
    e_ds = 72 * W * (G.abs() @ V[:, 0].abs().t()) + (G.abs() * e_out).sum(-1, keepdim=True) + (u + 2 * e) * (dp - delta).abs()
    if dtype == torch.float16:   # (ds is kept times 2^14 / (4 dim max|dout| max|v|) at least; half of fp16's smallest step)
        e_ds = e_ds + m * 2.0 ** -25 * 4 * dim * G.abs().max() * V.abs().max() / 2.0 ** 14
    limit = (e_ds + (m + 8) * W * (dp - delta).abs()).mean(-1)[..., None] * K[0, 0].abs() * dim ** -0.5
    worst = (dq.double().abs() / (limit * (1 + u) + 2.0 ** -25)).max().item()
    assert worst <= 1.0, worst
    # and the bound tells: delta made of the rounded out alone would leave more than it in many rows
    off = ((G @ (o.to(dtype).double() - o))[..., None] * K[0, 0] * dim ** -0.5).abs()
    assert ((off > limit).any(-1).double().mean() > 0.25).item()


@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("used", [[100, 3, 0, 57], [1, 1, 100, 99], [0, 0, 0, 1]])
def test_a_batched_cache_that_is_used_up_to_lengths_of_its_own(used, tokens):
    """Packed: a sequence for what is in use, and one of no queries for the room behind it, which may hold anything."""
    room, heads, kv_heads, dim, b = 100, 8, 2, 64, len(used)
    g = torch.Generator().manual_seed(tokens)
    q = torch.randn(b, tokens, heads, dim, generator=g).bfloat16().to(DEV)
    k, v = (torch.randn(b, room, kv_heads, dim, generator=g).bfloat16().to(DEV) for _ in range(2))
    at = torch.tensor(used, device=DEV)
    behind = torch.arange(room, device=DEV)[None] >= at[:, None]
    k[behind], v[behind] = math.nan, math.inf
    starts = torch.arange(b, device=DEV) * room
    cu_k = torch.cat([torch.stack([starts, starts + at], 1).flatten(), torch.tensor([b * room], device=DEV)]).int()
    cu = (torch.arange(2 * b + 1, device=DEV).add(1).div(2, rounding_mode="floor") * tokens).int()
    with torch.no_grad():
        out = attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), cu_seqlens=cu, cu_seqlens_k=cu_k).view_as(q)
    for i, n in enumerate(used):
        want, bound = exact(q[i], k[i, :n], v[i, :n], torch.zeros_like(q[i]), [(tokens, n)])
        near(out[i], want[0], bound[0], f"sequence {i}")
