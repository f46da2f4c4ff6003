"""Rows of attention whose scores are all minus infinity: the softmax of such a row is 0 / 0, so its output and its gradients are NaN, unlike those of a row that sees no key.

A key that scores minus infinity beside others which do not counts nothing.  Bounds are those of attention elsewhere (test_gpu_attention.py)."""
import math

import pytest
import torch
from test_gpu_attention import DEV, exact, inputs, near, offsets, step

from nanotron_amd.nn import attention

pytestmark = pytest.mark.gpu
E = 5   # the element of a head that an infinity is in


def hit_rows(q, k, rows, how, heads):
    """Every key of these rows scores minus infinity: an infinity in q against a negative element of every key, or a product beyond fp32."""
    q, k = q.clone(), k.clone()
    k[..., E] = -1.0
    for r in rows:
        q[r, heads, E] = math.inf
    if how == "overflow":
        k[..., E] = -(2.0 ** 100)
        q[..., E] = 0.0
        for r in rows:
            q[r, heads, E] = 2.0 ** 100
    return q, k


def check(q, k, v, do, lengths, rows, heads, causal, **kw):
    """(queries, keys) of the sequences; `rows` of `heads` are the bad ones."""
    out, dq, dk, dv = step(q, k, v, do, causal=causal, **kw)
    clean = q.clone()
    for r in rows:
        clean[r, heads] = 0.0
    want, bound = exact(clean, k, v, do, lengths, causal)
    hit = torch.zeros(q.shape, dtype=torch.bool, device=DEV)
    seen = torch.zeros(k.shape, dtype=torch.bool, device=DEV)
    group, a, b = q.shape[1] // k.shape[1], 0, 0
    for n, m in lengths:
        for r in rows:
            last = m - n + r - a if causal else m - 1
            if a <= r < a + n and last >= 0:
                for h in heads:
                    hit[r, h] = True
                    seen[b:b + last + 1, h // group] = True
        a, b = a + n, b + m
    for got, i, at, name in ((out, 0, hit, "out"), (dq, 1, hit, "dq"), (dk, 2, seen, "dk"), (dv, 3, seen, "dv")):
        assert torch.isnan(got[at]).all(), name
        near(got[~at], want[i][~at], bound[i][~at], name)
    with torch.no_grad():
        again = attention(q, k, v, causal=causal, **kw)
    assert torch.isnan(again[hit]).all()
    near(again[~hit], want[0][~hit], bound[0][~hit], "out without gradients")


HOW = [(torch.bfloat16, "infinity"), (torch.float16, "infinity"), (torch.bfloat16, "overflow")]


@pytest.mark.parametrize("dtype, how", HOW)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_of_one_sequence(dim, causal, dtype, how):
    """Tiles of 128 rows of a head: the first row, which sees one key, rows in whole and in masked tiles."""
    q, k, v, do = inputs(333, 2, 2, dim, dtype, seed=2)
    rows, heads = [0, 70, 200], [1]
    check(*hit_rows(q, k, rows, how, heads), v, do, [(333, 333)], rows, heads, causal)


@pytest.mark.parametrize("dtype, how", HOW)
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_packed_sequences(causal, dtype, how):
    """Tiles of 32 rows of four heads of a group, and rows in front of the first key, which see nothing and stay 0."""
    lengths = [(20, 20), (9, 4), (31, 90), (5, 0), (1, 1)]
    n, m = (sum(x[i] for x in lengths) for i in range(2))
    q, k, v, do = inputs(n, 8, 2, 64, dtype, keys=m, seed=3)
    rows, heads = [0, 7, 20, 26, 40, 59, 62, n - 1], [0, 5]
    check(*hit_rows(q, k, rows, how, heads), v, do, lengths, rows, heads, causal, cu_seqlens=offsets(lengths), cu_seqlens_k=offsets(lengths, 1))


@pytest.mark.parametrize("dtype, how", HOW)
@pytest.mark.parametrize("tokens, keys", [(1, 1), (1, 40), (3, 500), (1, 700), (4, 5000), (5, 2), (100, 3000), (20, 4096)])
def test_rows_over_a_cache(tokens, keys, dtype, how):
    """A few tokens, whose keys are cut between waves and workgroups, and more of them, whose keys are cut between workgroups."""
    b, heads, kv_heads, dim = 2, 8, 2, 64
    g = torch.Generator().manual_seed(tokens + keys)
    q = torch.randn(b * tokens, heads, dim, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(b * keys, kv_heads, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    rows, bad = sorted({0, tokens - 1, b * tokens - 1}), [1, 6]
    q, k = hit_rows(q, k, rows, how, bad)
    clean = q.clone()
    for r in rows:
        clean[r, bad] = 0.0
    want, bound = exact(clean, k, v, torch.zeros_like(q), [(tokens, keys)] * b)
    hit = torch.zeros(q.shape, dtype=torch.bool, device=DEV)
    for r in rows:
        if keys - tokens + r % tokens >= 0:
            for h in bad:
                hit[r, h] = True
    with torch.no_grad():
        out = attention(q.view(b, tokens, heads, dim), k.view(b, keys, kv_heads, dim), v.view(b, keys, kv_heads, dim)).flatten(0, 1)
    assert torch.isnan(out[hit]).all()
    near(out[~hit], want[0][~hit], bound[0][~hit], "out")


@pytest.mark.parametrize("tokens, keys, lost", [(1, 40, 32), (1, 40, 39), (1, 2000, 1500), (3, 2000, 1990), (100, 3000, 2048), (100, 3000, 1), (200, 200, 64)])
def test_keys_that_score_minus_infinity_beside_others_count_nothing(tokens, keys, lost):
    """The first `lost` keys score minus infinity for every query: whole runs of keys, or parts of one."""
    b, heads, kv_heads, dim = 2, 4, 2, 64
    g = torch.Generator().manual_seed(keys + lost)
    q = torch.randn(b, tokens, heads, dim, generator=g).bfloat16().to(DEV)
    k, v = (torch.randn(b, keys, kv_heads, dim, generator=g).bfloat16().to(DEV) for _ in range(2))
    q[..., E], k[..., E] = 2.0 ** 100, 0.0
    k[:, :lost, :, E] = -(2.0 ** 100)
    kept = [t[:, lost:].flatten(0, 1).contiguous() for t in (k, v)]
    clean = q.clone()
    clean[..., E] = 0.0
    clean = clean.flatten(0, 1)
    want, bound = exact(clean, *kept, torch.zeros_like(clean), [(tokens, keys - lost)] * b, causal=False)
    with torch.no_grad():
        near(attention(q, k, v, causal=False).flatten(0, 1), want[0], bound[0], "out")
