"""The operators of a decoder layer together, as a model uses them, against the same layer in 64 bits; and the example that trains one.

Tolerance of the layer: in a chain of n operators whose outputs are rounded to 16 bits, half a step of u = 2^-8 each, an operator adds u of its output
in the 2-norm at most and hands on what it was given times its condition, here 2 at most (a norm, a rotation, a mean of values, a product with a
matrix of random signs): 12 operators, forward and backward, 24 u = 0.094 on the way to a gradient, 0.047 to an output."""
import os
import sys

import pytest
import torch

from nanotron_amd.nn import RotaryEmbedding, attention, residual_rms_norm, rms_norm

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HIDDEN, HEADS, KV, DIM = 256, 8, 2, 32


def weights(dtype):
    g = torch.Generator().manual_seed(0)

    def matrix(n, m):
        return (torch.randn(n, m, generator=g) * m ** -0.5).bfloat16().to(DEV, dtype)

    w = dict(qkv=matrix((HEADS + 2 * KV) * DIM, HIDDEN), out=matrix(HIDDEN, HIDDEN), up=matrix(2 * HIDDEN, HIDDEN), down=matrix(HIDDEN, 2 * HIDDEN))
    for k in ("norm", "mlp_norm", "post", "gate"):
        w[k] = (1 + 0.2 * torch.randn(HIDDEN, generator=g)).bfloat16().to(DEV, dtype)
    return w


def layer(x, h, w, positions, cu, rotate):
    """What a block hands on: the MLP's output and the stream."""
    y, h = residual_rms_norm(x, h, w["norm"])
    q, k, v = (y @ w["qkv"].t()).unflatten(-1, (-1, DIM)).split([HEADS, KV, KV], 1)
    q, k = rotate(q, k, positions)
    a = attention(q, k, v, cu_seqlens=cu).flatten(1)
    y, h = residual_rms_norm(a @ w["out"].t(), h, w["mlp_norm"], post_weight=w["post"], gate=w["gate"], residual_scale=0.5)
    return torch.relu(y @ w["up"].t()) @ w["down"].t(), h


def plain_layer(x, h, w, positions, lengths, frequencies):
    def norm(t, weight):
        return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight

    def turn(t):
        angle = positions.double()[:, None, None] * frequencies
        a, b = t[..., :DIM // 2], t[..., DIM // 2:]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    h = h + x
    q, k, v = (norm(h, w["norm"]) @ w["qkv"].t()).unflatten(-1, (-1, DIM)).split([HEADS, KV, KV], 1)
    q, k = turn(q), turn(k)
    out, at = [], 0
    for n in lengths:
        s = slice(at, at + n)
        at += n
        p = torch.einsum("ihd,jhd->hij", q[s], k[s].repeat_interleave(HEADS // KV, 1)) * DIM ** -0.5
        p = torch.softmax(p.masked_fill(torch.ones(n, n, device=p.device).triu(1).bool(), -torch.inf), -1)
        out.append(torch.einsum("hij,jhd->ihd", p, v[s].repeat_interleave(HEADS // KV, 1)))
    h = 0.5 * h + w["gate"] * norm(torch.cat(out).flatten(1) @ w["out"].t(), w["post"])
    return torch.relu(norm(h, w["mlp_norm"]) @ w["up"].t()) @ w["down"].t(), h


def test_layer_against_64_bits():
    lengths = [50, 1, 129, 77]
    n = sum(lengths)
    positions = torch.cat([torch.arange(x) for x in lengths]).to(DEV)
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(1)
    x, h, dy, dh = (torch.randn(n, HIDDEN, generator=g).bfloat16().to(DEV) for _ in range(4))
    rotate = RotaryEmbedding(DIM, device=DEV)
    w = {k: v.requires_grad_(True) for k, v in weights(torch.bfloat16).items()}
    full = {k: v.detach().double().requires_grad_(True) for k, v in w.items()}
    leaves, twins = [t.requires_grad_(True) for t in (x, h)], [t.detach().double().requires_grad_(True) for t in (x, h)]
    got = layer(*leaves, w, positions, cu, rotate)
    want = plain_layer(*twins, full, positions, lengths, rotate.frequencies)
    grads = torch.autograd.grad(got, [*leaves, *w.values()], (dy, dh))
    exact = torch.autograd.grad(want, [*twins, *full.values()], (dy.double(), dh.double()))
    for name, a, b, bound in [("y", got[0], want[0], 0.047), ("h", got[1], want[1], 0.047), *((k, a, b, 0.094) for k, a, b in zip(["x", "h", *w], grads, exact))]:
        off = ((a.detach().double() - b).norm() / b.norm()).item()
        assert off <= bound, (name, off)


def test_one_token_after_another_is_the_whole_prompt():
    """Evaluation token by token over a cache gives what the whole prompt gives at once."""
    n = 40
    rotate = RotaryEmbedding(DIM, device=DEV)
    qkv = torch.randn(2, n, HEADS + 2 * KV, DIM, device=DEV).bfloat16()
    q, k, v = qkv.split([HEADS, KV, KV], 2)
    with torch.no_grad():
        rq, rk = rotate(q, k, torch.arange(n, device=DEV))
        want = attention(rq, rk, v)
        cache = torch.zeros(2, 2, 64, KV, DIM, device=DEV, dtype=torch.bfloat16)
        for i in range(n):
            a, b = rotate(q[:, i:i + 1], k[:, i:i + 1], torch.tensor([i], device=DEV))
            cache[0][:, i:i + 1], cache[1][:, i:i + 1] = b, v[:, i:i + 1]
            one = attention(a, cache[0][:, :i + 1], cache[1][:, :i + 1])
            # two orders of the same sums, the numerators rounded to 16 bits in each: 2^-8 of a mean of values apart, and one rounding each
            assert (one - want[:, i:i + 1]).abs().max() <= 4 * 2.0 ** -8 * v.abs().max()
            assert torch.equal(a, rq[:, i:i + 1]) and torch.equal(b, rk[:, i:i + 1])


def test_norm_in_front_of_a_model_is_that_of_a_first_block():
    x = torch.randn(30, HIDDEN, device=DEV).bfloat16()
    w = torch.ones(HIDDEN, device=DEV)
    assert torch.equal(rms_norm(x, w), residual_rms_norm(x, torch.zeros_like(x), w)[0])


def test_example_runs_and_every_parameter_has_a_gradient():
    import train_language_model as example

    losses = example.train(3, 128, 2, 500, 256, heads=4, kv_heads=2)
    assert len(losses) == 3 and all(0 < x < 20 for x in losses)
    torch.manual_seed(0)
    model = example.LanguageModel(500, 128, 2, heads=4, kv_heads=2)
    tokens, labels = next(example.batches(500, 64, 4, "cuda", 1))
    model(tokens, labels).backward()
    opt = example.optimizer_of(model, 1e-3, 8)
    grads = [opt.grad_of(p, copy).as_subclass(torch.Tensor).float() for p, copy in opt.params_and_copies()]
    assert len(grads) == len(list(model.parameters()))
    for g in grads:
        assert torch.isfinite(g).all() and g.abs().max() > 0, g.shape
