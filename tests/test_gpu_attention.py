"""Attention against its formulas in 64 bits.

Tolerances, with u = 2^-8 (bf16) or 2^-11 (fp16), half a step of what is rounded to 16 bits, and w = 2^-24.  A score is a sum of D products in fp32:
off by (D + 4) w c sum|q||k| in the exponent, and exponential, maximum and logarithm bring 16 w each way, so the softmax p and what it is
divided by are off by e = 2 (D + 4) w c max sum|q||k| + (n + 64) w relative, n keys being added up.  The numerators are rounded once for the
product: out is off by (u + e) p|v|, and u |out| for its own rounding.  dv by (u + e) p^T|dout| and its rounding.  delta is made of the rounded
out: off by |dout| (what out is off by); dout v^T by D w |dout||v|; ds = p (..) by p times both and (u + 2 e) |ds|, of which dq and dk are
sums with |k| and |q|, n more w for adding up.  fp16 has a smallest step besides, 2^-25 half of it: of p, kept below its row's maximum times 2^8 at most
(forward) or times 2^8 (backward), and of ds, kept times 2^14 / (4 D max|dout| max|v|) at least.  And fp32's normal numbers end at 2^-126: a p or ds
below that may count as 0 (a score 90 standard deviations below its row's maximum has such a p, and its key, if no other row attends to it, a gradient
of that size)."""
import math

import pytest
import torch

from nanotron_amd.nn import attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W = 2.0 ** -24


def exact_one(q, k, v, do, scale, causal, u, tiny):
    """One head of one sequence, [rows, dim] in 64 bits: (out, dq, dk, dv) and what each may be off by before its own rounding."""
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    s = q @ k.t() * scale
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = torch.arange(m, device=q.device)[None] <= torch.arange(m - n, m, device=q.device)[:, None]
    any_ = seen.any(-1, keepdim=True)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.where(any_, torch.softmax(torch.where(any_, s, 0.0), -1), 0.0).masked_fill(~seen, 0.0)
    qk = ((q.abs() @ k.abs().t()).masked_fill(~seen, 0.0).amax(-1, keepdim=True) if m else torch.zeros(n, 1, device=q.device, dtype=q.dtype)) * scale
    e = 2 * (d + 4) * W * 1.45 * qk + (m + 64) * W
    o = p @ v
    low = 2.0 ** -126 * seen.double()
    step = tiny * seen.double() + low   # of a numerator, beside the sum, which is 1 or more
    eo = (u + e) * (p @ v.abs()) + step @ v.abs()
    dv = p.t() @ do
    edv = ((u + e) * p + tiny / 256 * seen.double() + low).t() @ do.abs()
    dp = do @ v.t()
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = d * W * (do.abs() @ v.abs().t()) + (do.abs() * (eo + u * (o.abs() + eo) + d * W * o.abs())).sum(-1, keepdim=True)
    lift = 2.0 ** 14 / (4 * d * max(1e-30, do.abs().max().item() if n else 0) * max(1e-30, v.abs().max().item() if m else 0))
    eds = p * off + (u + 2 * e) * ds.abs() + tiny * seen.double() / lift + low * (1 + dp.abs() + delta.abs())
    more = (max(n, m) + 8) * W
    return (o, ds @ k * scale, ds.t() @ q * scale, dv), (eo, (eds + more * ds.abs()) @ k.abs() * scale, (eds + more * ds.abs()).t() @ q.abs() * scale, edv + more * p.t() @ do.abs())


def exact(q, k, v, do, lengths, causal=True, scale=None):
    """q [tokens, heads, dim] and the others; lengths: (queries, keys) of the sequences, end to end."""
    u, tiny = U[q.dtype], 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    args = [t.double() for t in (q, k, v, do)]
    want, bound = ([torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, q, k, v)] for _ in range(2))
    a = b = 0
    for n, m in lengths:
        if n and m:
            for h in range(q.shape[1]):
                j = h // group
                r, x = exact_one(args[0][a:a + n, h], args[1][b:b + m, j], args[2][b:b + m, j], args[3][a:a + n, h], scale, causal, u, tiny)
                for t, y in ((want, r), (bound, x)):
                    t[0][a:a + n, h] += y[0]
                    t[1][a:a + n, h] += y[1]
                    t[2][b:b + m, j] += y[2]
                    t[3][b:b + m, j] += y[3]
        a, b = a + n, b + m
    return want, bound


def near(got, want, bound, name):
    u = U[got.dtype]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[got.dtype]
    assert torch.isfinite(got).all(), name
    off = (got.double() - want).abs()
    limit = bound + u * (want.abs() + bound) + tiny
    worst = (off / limit.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times what it may be off"


def inputs(tokens, heads, kv_heads, dim, dtype, keys=None, seed=0, gradient=0.1):
    g = torch.Generator().manual_seed(seed)
    keys = tokens if keys is None else keys

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)

    return normal(tokens, heads, dim, std=1.5), normal(keys, kv_heads, dim), normal(keys, kv_heads, dim), normal(tokens, heads, dim, std=gradient)


def offsets(lengths, which=0):
    at = [0]
    for x in lengths:
        at.append(at[-1] + (x[which] if isinstance(x, tuple) else x))
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def step(q, k, v, do, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention(q, k, v, **kw)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))


def check(q, k, v, do, lengths, causal=True, scale=None, **kw):
    got = step(q, k, v, do, causal=causal, scale=scale, **kw)
    want, bound = exact(q, k, v, do, lengths, causal, scale)
    for o, a, e, n in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        assert o.shape == a.shape and o.dtype == q.dtype and o.is_contiguous()
        near(o, a, e, n)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 8, 72, 96, 104])
@pytest.mark.parametrize("causal", [True, False])
def test_one_sequence(dtype, dim, causal):
    q, k, v, do = inputs(333, 4, 2, dim, dtype)
    check(q, k, v, do, [(333, 333)], causal)


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257])
def test_lengths(length):
    q, k, v, do = inputs(length, 2, 1, 64, torch.bfloat16, seed=length)
    check(q, k, v, do, [(length, length)])


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 2), (8, 1), (6, 3), (5, 1)])
def test_heads(heads, kv_heads):
    q, k, v, do = inputs(150, heads, kv_heads, 64, torch.bfloat16)
    check(q, k, v, do, [(150, 150)])


PACKED = [[1], [5, 7, 1, 0, 3], [0, 0, 200], [200, 0, 0], [64, 64, 64], [128, 1, 127, 130], [1] * 70, [300, 17, 1, 90]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", PACKED)
def test_packed(lengths, causal):
    n = sum(lengths)
    q, k, v, do = inputs(n, 4, 2, 128, torch.bfloat16, seed=n)
    check(q, k, v, do, [(x, x) for x in lengths], causal, cu_seqlens=offsets(lengths))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", [[(3, 70), (1, 1), (40, 40)], [(70, 3), (5, 200), (0, 9), (9, 0), (130, 129)], [(1, 300)], [(300, 1)], [(0, 4), (4, 0)]])
def test_more_or_fewer_keys(lengths, causal):
    """Causal rows in front of the first key see nothing: 0, and no gradient."""
    n, m = (sum(x[i] for x in lengths) for i in range(2))
    q, k, v, do = inputs(n, 4, 2, 64, torch.bfloat16, keys=m, seed=m)
    got = check(q, k, v, do, lengths, causal, cu_seqlens=offsets(lengths), cu_seqlens_k=offsets(lengths, 1))
    a = 0
    for x, y in lengths:
        if causal and x > y:
            assert not got[0][a:a + x - y].any() and not got[1][a:a + x - y].any()
        a += x


@pytest.mark.parametrize("tokens,keys", [(1, 1), (1, 7), (1, 300), (1, 5000), (3, 1000), (8, 8), (8, 33), (9, 1), (17, 900), (100, 3000), (65, 64)])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 80)])
def test_batches(tokens, keys, dtype, dim):
    """A batch of equal lengths, fewer or more rows than one tile, keys the first part of a cache."""
    b, heads, kv = 3, 8, 2
    g = torch.Generator().manual_seed(tokens + keys)
    q = (1.5 * torch.randn(b, tokens, heads, dim, generator=g)).to(dtype).to(DEV)
    k, v = ((torch.randn(b, keys + 5, kv, dim, generator=g)).to(dtype).to(DEV)[:, :keys] for _ in range(2))
    do = torch.randn(b, tokens, heads, dim, generator=g).mul_(0.1).to(dtype).to(DEV)
    got = step(q, k, v, do)
    flat = [t.reshape(-1, *t.shape[2:]) for t in (q, k, v, do)]
    want, bound = exact(*flat, [(tokens, keys)] * b)
    for o, a, e, n in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        near(o.flatten(0, 1), a, e, n)
    with torch.no_grad():
        assert torch.equal(attention(q, k, v), got[0])


def test_many_sequences_of_a_batch():
    q = torch.randn(200, 1, 4, 64, device=DEV).bfloat16()
    k, v = (torch.randn(200, 40, 1, 64, device=DEV).bfloat16() for _ in range(2))
    want, bound = exact(*(t.flatten(0, 1) for t in (q, k, v, q)), [(1, 40)] * 200)
    with torch.no_grad():
        near(attention(q, k, v).flatten(0, 1), want[0], bound[0], "out")


def test_long_rows():
    q, k, v, do = inputs(3000, 2, 1, 128, torch.bfloat16)
    check(q, k, v, do, [(3000, 3000)])


@pytest.mark.parametrize("scale", [1.0, 0.01, 7.5])
def test_scales(scale):
    q, k, v, do = inputs(200, 2, 2, 64, torch.bfloat16)
    check(q, k, v, do, [(200, 200)], scale=scale)


def test_large_scores():
    """Scores of hundreds: the softmax is a choice of one key, and nothing overflows."""
    q, k, v, do = inputs(300, 2, 1, 128, torch.bfloat16)
    check(q * 16, k * 4, v, do, [(300, 300)])
    # in rising order, so that the running maximum is raised again and again
    order = (q[:, 0].float() @ k[:, 0].float().t()).sum(0).argsort()
    check(q * 16, k[order].contiguous(), v[order].contiguous(), do, [(300, 300)], causal=False)


@pytest.mark.parametrize("gradient", [1e-6, 1e-3, 100.0])
def test_small_and_large_gradients_of_fp16(gradient):
    q, k, v, do = inputs(700, 2, 1, 64, torch.float16, gradient=gradient)
    check(q, k, v, do, [(700, 700)])


def test_strided_views():
    """Parts of one linear's output, heads in front of tokens, rows that repeat."""
    qkv = torch.randn(260, 12, 64, device=DEV).bfloat16()
    do = torch.randn(260, 8, 64, device=DEV).bfloat16()
    parts = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    check(*parts, do, [(260, 260)])
    dense = [t.contiguous() for t in parts]
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in dense]
    for a, b in zip(step(*dense, do), step(*turned, do.transpose(0, 1).contiguous().transpose(0, 1))):
        assert torch.equal(a, b)
    # off 16-byte boundaries, an odd distance apart: copied
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in dense]
    assert all(t.stride(1) == 67 for t in odd)
    for a, b in zip(step(*dense, do), step(*odd, do)):
        assert torch.equal(a, b)
    one = dense[1][:1].expand(260, 2, 64)
    check(dense[0], one, one, do, [(260, 260)])


def test_gradient_that_is_broadcast():
    q, k, v, _ = inputs(130, 4, 2, 64, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    a = torch.autograd.grad(attention(*leaves).sum(), leaves)
    b = torch.autograd.grad(attention(*leaves), leaves, torch.ones_like(q))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    attention(*leaves).float().square().sum().backward()
    assert all(t.grad is not None and torch.isfinite(t.grad).all() for t in leaves)


@pytest.mark.parametrize("leaf", [0, 1, 2])
def test_one_gradient_at_a_time(leaf):
    q, k, v, do = inputs(140, 4, 2, 64, torch.bfloat16)
    every = step(q, k, v, do)
    t = (q, k, v)[leaf].requires_grad_(True)
    assert torch.equal(torch.autograd.grad(attention(q, k, v), t, do)[0], every[leaf + 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_seen_does_not_arrive(dtype, bad):
    """NaN and infinities in rows of no sequence, in the sequence behind, and in tokens to come."""
    lengths, pad = [100, 90, 60], 40
    n = sum(lengths)
    q, k, v, do = inputs(n, 4, 2, 64, dtype, seed=3)
    clean = step(q, k, v, do, cu_seqlens=offsets(lengths))
    spoilt = [torch.cat([t, torch.full((pad, *t.shape[1:]), bad, dtype=dtype, device=DEV)]) for t in (q, k, v, do)]
    got = step(*spoilt, cu_seqlens=offsets(lengths))
    for a, b, name in zip(got, clean, ("out", "dq", "dk", "dv")):
        assert torch.equal(a[:n], b), name
        assert not a[n:].any(), name
    # sequence 1 spoilt: 0 and 2 are as they were
    for which in range(4):
        args = [t.clone() for t in (q, k, v, do)]
        args[which][100:190] = bad
        for a, b in zip(step(*args, cu_seqlens=offsets(lengths)), clean):
            assert torch.equal(a[:100], b[:100]) and torch.equal(a[190:], b[190:])
    # a token to come: rows in front of it are as they were, forward
    for at in (99, 50, 33, 64):
        for which in (1, 2):
            args = [t.clone() for t in (q, k, v)]
            args[which][at] = bad
            with torch.no_grad():
                out = attention(*args, cu_seqlens=offsets(lengths))
            assert torch.isfinite(out[:at]).all()
            near(out[:at], clean[0][:at].double(), (clean[0][:at].double().abs() + 1e-3) * 4 * U[dtype], "rows in front")
            assert not torch.isfinite(out[at]).any() or which == 1
            assert torch.equal(out[100:], clean[0][100:])


@pytest.mark.parametrize("dtype, dim, heads, kv_heads", [(torch.bfloat16, 128, 4, 2), (torch.float16, 80, 2, 2), (torch.float16, 64, 6, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_bad_values_in_several_tiles(dtype, dim, heads, kv_heads, causal):
    """Values that are not finite, in tiles of several steps, reach the rows that see them and the elements that they are in, and nothing else."""
    lengths, rows = [333, 5, 270], (333 + 5 + 64, 333 + 5 + 200)
    n, first = sum(lengths), 338
    q, k, v, do = inputs(n, heads, kv_heads, dim, dtype, seed=8)
    cu = offsets(lengths)
    want, bound = exact(q, k, v, do, [(x, x) for x in lengths], causal)

    def same(got, name, at):
        i = ("out", "dq", "dk", "dv").index(name)
        near(got[at], want[i][at], bound[i][at], name)

    # a value: its element of the rows behind it, of the heads that share it; gradients of the rows in front of it
    bad = v.clone()
    bad[rows[0], 0, 5], bad[rows[1], kv_heads - 1, dim - 1] = math.inf, math.nan
    out, dq, dk, dv = step(q, k, bad, do, cu_seqlens=cu, causal=causal)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    group = heads // kv_heads
    hit[rows[0] if causal else first:, :group, 5] = True
    hit[rows[1] if causal else first:, heads - group:, dim - 1] = True
    assert torch.equal(~torch.isfinite(out), hit)
    same(out, "out", ~hit)
    same(dv[:first], "dv", slice(0, first))
    if causal:
        assert torch.isfinite(dq[:rows[0]]).all()
        same(dq, "dq", slice(first, rows[0]))
    # a gradient: its element of the values that it saw, in the heads' own
    bad = do.clone()
    bad[rows[0], 0, 3] = bad[rows[1], 0, 3] = math.nan
    out, dq, dk, dv = step(q, k, v, bad, cu_seqlens=cu, causal=causal)
    hit = torch.zeros(dv.shape, dtype=torch.bool, device=DEV)
    hit[first:rows[1] + 1 if causal else n, 0, 3] = True
    assert torch.equal(~torch.isfinite(dv), hit)
    same(dv, "dv", ~hit)
    hit = torch.zeros(dq.shape, dtype=torch.bool, device=DEV)
    hit[rows[0], 0] = hit[rows[1], 0] = True
    assert torch.equal(~torch.isfinite(dq), hit)
    hit = torch.zeros(dk.shape, dtype=torch.bool, device=DEV)
    hit[first:rows[1] + 1 if causal else n, 0] = True
    assert torch.equal(~torch.isfinite(dk), hit)
    # a key: the queries that see it
    bad = k.clone()
    bad[rows[1], 0, 7] = math.nan
    out, dq, dk, dv = step(q, bad, v, do, cu_seqlens=cu, causal=causal)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[rows[1] if causal else first:, :group] = True
    assert torch.equal(~torch.isfinite(out), hit) and torch.equal(~torch.isfinite(dq), hit)
    same(out, "out", ~hit)


@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 80)])
@pytest.mark.parametrize("keys", [40, 700])
def test_bad_values_behind_a_few_tokens(dtype, dim, keys):
    """Six tokens of a batch over a cache whose last values are not finite: tokens in front of these see nothing of them."""
    g = torch.Generator().manual_seed(keys)
    q, k, v = (torch.randn(3, n, h, dim, generator=g).to(dtype).to(DEV) for n, h in ((6, 4), (keys, 2), (keys, 2)))
    with torch.no_grad():
        bad = v.clone()
        bad[1, keys - 3, 1, 4], bad[1, keys - 2, 0, 9] = math.inf, math.nan
        out = attention(q, k, bad)
        hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
        hit[1, 3:, 2:, 4] = True
        hit[1, 4:, :2, 9] = True
        assert torch.equal(~torch.isfinite(out), hit)
        flat = [t.flatten(0, 1) for t in (q, k, v)]
        want, bound = exact(*flat, torch.zeros_like(flat[0]), [(6, keys)] * 3)
        near(out[~hit], want[0].view_as(out)[~hit], bound[0].view_as(out)[~hit], "elements beside")
        bad = k.clone()
        bad[2, keys - 1] = math.nan
        out = attention(q, bad, v)
        assert torch.isfinite(out[:2]).all() and torch.isfinite(out[2, :5]).all() and torch.isnan(out[2, 5]).all()


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_gradients_beside_a_bad_row(which):
    """A row that is not finite spoils the gradients that the formula says, in its tile too, and no others: keys behind a bad query see nothing of it,
    nor do queries in front of a bad key."""
    n, at = 64, 20
    q, k, v, do = inputs(n, 1, 1, 64, torch.bfloat16, seed=4)
    clean = step(q, k, v, do)
    args = [t.clone() for t in (q, k, v, do)]
    args[which][at] = math.nan
    got = step(*args)
    if which in (0, 3):   # a query: its own dq, and dk and dv of the keys that it sees
        assert torch.isfinite(got[1][:at]).all() and torch.isfinite(got[1][at + 1:]).all()
        for g, c in zip(got[2:], clean[2:]):
            assert torch.isfinite(g[at + 1:]).all()
            near(g[at + 1:], c[at + 1:].double(), (c[at + 1:].double().abs() + 1e-3) * 4 * U[g.dtype], "keys behind")
    else:                 # a key: dq of the queries that see it
        assert torch.isfinite(got[1][:at]).all()
        near(got[1][:at], clean[1][:at].double(), (clean[1][:at].double().abs() + 1e-3) * 4 * U[q.dtype], "queries in front")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_lose_little_beyond_their_own_roundings(dtype):
    """In the 2-norm a rounding of values of any significand costs 0.41 u (2 u / sqrt(12), and sqrt(1/2) for significands between 1 and 2).  dq and
    dk are rounded, and so is ds: 0.58 u.  What else there is, out's own error in the subtracted sums first of all, is to be less than one
    rounding: sqrt(3) 0.41 u = 0.71 u.  (With the sums made of the rounded out it is more in sequences as short as these.)"""
    lengths = [7, 20, 33, 64, 15, 90, 41, 5]
    n = sum(lengths)
    q, k, v, do = inputs(n, 8, 4, 64, dtype, seed=11)
    got = step(q, k, v, do, cu_seqlens=offsets(lengths))
    want, _ = exact(q, k, v, do, [(x, x) for x in lengths])
    for o, a, name in zip(got, want, ("out", "dq", "dk", "dv")):
        off = ((o.double() - a).norm() / a.norm()).item()
        assert off <= 3 ** 0.5 * 0.41 * U[dtype], (name, off / U[dtype])


def test_offsets_that_are_wrong_stay_inside():
    """Offsets behind the rows that there are, or below zero, count as the nearest inside; rows of no sequence are zeros."""
    q, k, v, do = inputs(100, 2, 1, 64, torch.bfloat16)
    cu = torch.tensor([-5, 40, 1000], dtype=torch.int32, device=DEV)
    for a, b in zip(step(q, k, v, do, cu_seqlens=cu), step(q, k, v, do, cu_seqlens=offsets([40, 60]))):
        assert torch.equal(a, b)
    cu = torch.tensor([30, 60, 80], dtype=torch.int32, device=DEV)
    got = step(q, k, v, do, cu_seqlens=cu)
    inner = step(*(t[30:80].contiguous() for t in (q, k, v, do)), cu_seqlens=offsets([30, 20]))
    for a, b in zip(got, inner):
        assert not a[:30].any() and not a[80:].any() and torch.equal(a[30:80], b)


def test_nothing_to_do():
    q, k, v, do = inputs(0, 4, 2, 64, torch.bfloat16, keys=5)
    got = step(q, k, v, do)
    assert got[0].shape == (0, 4, 64) and not got[2].any() and not got[3].any()
    q, k, v, do = inputs(6, 4, 2, 64, torch.bfloat16, keys=0)
    got = step(q, k, v, do)
    assert not got[0].any() and not got[1].any() and got[2].shape == (0, 2, 64)
    e = torch.zeros(0, 3, 4, 64, device=DEV, dtype=torch.bfloat16)
    assert attention(e, e, e).shape == e.shape


def test_same_bits_again():
    q, k, v, do = inputs(900, 8, 2, 128, torch.bfloat16)
    cu = offsets([400, 37, 463])
    first = step(q, k, v, do, cu_seqlens=cu)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step(q, k, v, do, cu_seqlens=cu)))


def test_gradient_against_differences():
    """The forward pass in 64 bits, differenced: an independent statement of the gradients, which the kernels' then meet within 16-bit rounding."""
    q, k, v, do = inputs(9, 2, 1, 16, torch.float16)
    got = step(q, k, v, do)[1:]
    full = [t.double() for t in (q, k, v)]

    def value(q, k, v):
        x = torch.einsum("ihd,jd->hij", q.cpu(), k[:, 0].cpu()) / 4.0
        x = x.masked_fill(torch.ones(9, 9).triu(1).bool(), -math.inf)
        return (torch.einsum("hij,jd->ihd", torch.softmax(x, -1), v[:, 0].cpu()) * do.double().cpu()).sum().item()

    h = 1e-5
    for i, g in enumerate(got):
        flat = full[i].view(-1)
        for at in range(0, flat.numel(), 7):
            keep = flat[at].item()
            flat[at] = keep + h
            up = value(*full)
            flat[at] = keep - h
            down = value(*full)
            flat[at] = keep
            assert abs((up - down) / (2 * h) - g.view(-1)[at].item()) < 4e-3 * g.abs().max().item() + 1e-6


def test_graph_replays():
    """Captured forward and backward, replayed with other inputs and eager calls between."""
    q, k, v, do = inputs(500, 4, 2, 64, torch.float16)
    cu = offsets([200, 300])
    static = [t.clone() for t in (q, k, v, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static, cu_seqlens=cu)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static, cu_seqlens=cu)
    for seed, lengths in ((5, [200, 300]), (6, [499, 1]), (7, [0, 500])):
        fresh = inputs(500, 4, 2, 64, torch.float16, seed=seed)
        for a, b in zip(static, fresh):
            a.copy_(b)
        cu.copy_(offsets(lengths))   # other lengths too: the device reads them
        graph.replay()
        torch.cuda.synchronize()
        want = step(*fresh, cu_seqlens=offsets(lengths))
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_two_graphs_of_one_token_over_a_cache():
    q = torch.randn(2, 1, 8, 128, device=DEV).bfloat16()
    cache = torch.randn(2, 4096, 2, 128, device=DEV).bfloat16()
    with torch.no_grad():
        graphs, outs = [], []
        for n in (4000, 1500):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                attention(q, cache[:, :n], cache[:, :n])
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(attention(q, cache[:, :n], cache[:, :n]))
            graphs.append(g)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(3):
            torch.cuda.synchronize()
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for n, o in zip((4000, 1500), outs):
                assert torch.equal(o, attention(q, cache[:, :n], cache[:, :n]))
            q.normal_()


def test_another_stream():
    q, k, v, do = inputs(400, 4, 2, 64, torch.bfloat16)
    want = step(q, k, v, do)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(q, k, v, do)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_twice_backward_and_inference():
    q, k, v, do = inputs(300, 4, 2, 80, torch.float16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    cu = offsets([120, 0, 180])
    out = attention(*leaves, cu_seqlens=cu)
    first = torch.autograd.grad(out, leaves, do, retain_graph=True)
    second = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.inference_mode():
        assert torch.equal(attention(*leaves, cu_seqlens=cu), out)
        few = attention(q[None, :1], k[None], v[None])
    near(few[0], attention(q[None, :1].detach(), k[None].detach(), v[None].detach())[0].double(), 0.0 * few[0].double(), "one token")


def test_a_cache_of_more_than_2_32_bytes():
    """One new token, and a few, over 9 million keys: all of them 0 but some far ones, so the softmax is known in closed form."""
    n, kv, dim = 9_000_000, 2, 128
    k, v = (torch.zeros(1, n, kv, dim, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    assert k.numel() * 2 > 1 << 32
    spots = torch.tensor([0, 5, 4_194_303, 4_194_304, 8_388_608, 8_500_001, n - 2], device=DEV)
    g = torch.Generator().manual_seed(0)
    k[:, spots] = torch.randn(1, len(spots), kv, dim, generator=g).mul_(2).bfloat16().to(DEV)
    v[:, spots] = torch.randn(1, len(spots), kv, dim, generator=g).bfloat16().to(DEV)
    for tokens in (1, 40):
        q = torch.randn(1, tokens, 4, dim, generator=g).mul_(2).bfloat16().to(DEV)
        with torch.no_grad():
            out = attention(q, k, v, causal=False)
        s = torch.einsum("ihd,jhd->hij", q[0].double().cpu(), k[0, spots].double().cpu().repeat_interleave(2, 1)) * dim ** -0.5
        e = torch.exp(s)
        total = e.sum(-1, keepdim=True) + (n - len(spots))
        far = v[0, spots].double().cpu().repeat_interleave(2, 1)
        want = torch.einsum("hij,jhd->ihd", e / total, far)
        # numerators rounded to 16 bits, a sum of nine million ones in fp32 (runs of 2^20 at most, joined: 2^-4 of one in each addition's rounding)
        bound = (U[q.dtype] + 2.0 ** -12) * torch.einsum("hij,jhd->ihd", e / total, far.abs())
        near(out[0].cpu(), want, bound, f"{tokens} tokens")


def test_rows_far_apart():
    """Rows 2^24 elements apart, the last ones more than 2^32 bytes from the first."""
    n, far = 140, 1 << 24
    room = torch.zeros(n * far, device=DEV, dtype=torch.bfloat16)
    assert room.numel() * 2 > 1 << 32
    q, k, v, do = inputs(n, 4, 2, 64, torch.bfloat16)
    at, views = 0, []
    for t in (q, k, v, do):
        view = room.as_strided(t.shape, (far, 64, 1), at)
        view.copy_(t)
        views.append(view)
        at += 4096
    for a, b in zip(step(*views), step(q, k, v, do)):
        assert torch.equal(a, b)
    # one step further apart: copied
    room = torch.zeros(4 * (far + 8), device=DEV, dtype=torch.bfloat16)
    view = room.as_strided((4, 4, 64), (far + 8, 64, 1), 0)
    view.copy_(q[:4])
    assert torch.equal(attention(view, k[:4], v[:4]), attention(q[:4], k[:4], v[:4]))


@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 2, 128), (6, 2, 64), (5, 1, 80), (12, 2, 64), (4, 4, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_tokens_over_caches_of_different_lengths(heads, kv_heads, dim, causal):
    """Packed sequences of a few queries each over keys of their own, and one of many queries between them, without gradients."""
    lengths = [(1, 900), (1, 1), (0, 50), (3, 0), (2, 65), (1, 2000), (33, 40), (1, 64), (7, 3), (90, 300), (1, 129), (1, 511), (1, 7), (1, 70), (2, 2), (1, 1)]
    for dtype in (torch.bfloat16, torch.float16):
        n, m = sum(a for a, _ in lengths), sum(b for _, b in lengths)
        q, k, v, do = inputs(n, heads, kv_heads, dim, dtype, keys=m, seed=heads)
        want, bound = exact(q, k, v, do, lengths, causal)
        with torch.no_grad():
            out = attention(q, k, v, cu_seqlens=offsets(lengths), cu_seqlens_k=offsets(lengths, 1), causal=causal)
        near(out, want[0], bound[0], "out")
        # a cache that is not finite (the one key of the second sequence) is that of its own queries
        bad = v.clone()
        bad[900] = math.nan
        with torch.no_grad():
            other = attention(q, k, bad, cu_seqlens=offsets(lengths), cu_seqlens_k=offsets(lengths, 1), causal=causal)
        rows = torch.arange(n, device=DEV) != 1
        assert torch.equal(other[rows], out[rows]) and not torch.isfinite(other[1]).any()
        # rows of no sequence
        pad = torch.full((40, heads, dim), math.inf, dtype=dtype, device=DEV)
        with torch.no_grad():
            more = attention(torch.cat([q, pad]), k, v, cu_seqlens=offsets(lengths), cu_seqlens_k=offsets(lengths, 1), causal=causal)
        near(more[:n], want[0], bound[0], "out")
        assert not more[n:].any()


def test_many_short_sequences():
    """More sequences than a workgroup of the plan has threads."""
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 4, (3000,), generator=g).tolist()
    n = sum(lengths)
    q, k, v, do = inputs(n, 2, 1, 64, torch.bfloat16)
    got = step(q, k, v, do, cu_seqlens=offsets(lengths))
    # one sequence under a mask of blocks is the same
    owner = torch.repeat_interleave(torch.arange(3000), torch.tensor(lengths)).to(DEV)
    at = torch.arange(n, device=DEV)
    seen = (owner[:, None] == owner[None]) & (at[None] <= at[:, None])
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    p = torch.softmax((torch.einsum("ihd,jd->hij", leaves[0], leaves[1][:, 0]) * 0.125).masked_fill(~seen, -math.inf), -1)
    want = torch.einsum("hij,jd->ihd", p, leaves[2][:, 0])
    exact_ = (want.detach(), *torch.autograd.grad(want, leaves, do.double()))
    for o, a, name in zip(got, exact_, ("out", "dq", "dk", "dv")):
        # (sequences of three: the bound of a rounding of every operand, twice)
        assert ((o.double() - a).norm() / a.norm()).item() < 4 * U[q.dtype], name


def test_sequences_of_every_length_beside_each_other():
    """1500 sequences of 0 to 140 rows and a few of many tiles: more than a lane of the plan's kernel each, of one tile and of several."""
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 141, (1500,), generator=g).tolist()
    lengths[7], lengths[1023], lengths[1024], lengths[1499] = 700, 1300, 129, 257
    n = sum(lengths)
    q, k, v, do = inputs(n, 1, 1, 64, torch.bfloat16, seed=6)
    cu = offsets(lengths)
    for causal in (True, False):
        check(q, k, v, do, [(x, x) for x in lengths], causal, cu_seqlens=cu)


def test_refusals():
    q, k, v, do = inputs(10, 4, 2, 64, torch.bfloat16)
    cu = offsets([4, 6])
    for e, args, kw in (
            (TypeError, (q.float(), k.float(), v.float()), {}), (TypeError, (q, k.half(), v), {}), (ValueError, (q, k, v[:5]), {}),
            (ValueError, (q[:, :3], k, v), {}), (ValueError, (q[..., :60], k[..., :60], v[..., :60]), {}), (ValueError, (q[0], k[0], v[0]), {}),
            (ValueError, (q, k, v), dict(scale=0.0)), (ValueError, (q, k, v), dict(scale=-1.0)), (TypeError, (q, k, v), dict(cu_seqlens=cu.long())),
            (ValueError, (q, k, v), dict(cu_seqlens=cu[:1])), (ValueError, (q, k, v), dict(cu_seqlens_k=cu)), (ValueError, (q, k, v), dict(cu_seqlens=cu.cpu())),
            (ValueError, (q, k, v), dict(cu_seqlens=cu, cu_seqlens_k=offsets([10]))), (ValueError, (q[:5], k, v), dict(cu_seqlens=cu)),
            (ValueError, (q[None], k[None], v[None]), dict(cu_seqlens=cu)), (ValueError, (torch.zeros(2, 2, 136, device=DEV, dtype=torch.bfloat16),) * 3, {}),
            (ValueError, (q[:, :0], k, v), {}), (ValueError, (q.cpu(), k, v), {})):
        with pytest.raises(e):
            attention(*args, **kw)
    leaf = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(attention(leaf, k, v).sum(), leaf, create_graph=True)
