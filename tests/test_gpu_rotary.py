"""Rotary positions against complex multiplication in 64 bits.

Tolerances, with w = 2^-24: the turns are exact to 2^-52 of themselves, their fraction is rounded to fp32 (an angle off by 2 pi w / 2),
sine and cosine are good to 4 w, scale, the two products and their sum bring another 4 w: 16 w (|a| + |b|) |scale| in all, before the rounding to the type."""
import math

import pytest
import torch

from nanotron_amd.nn import RotaryEmbedding, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W = 2.0 ** -24


def exact(x, positions, frequencies, interleaved, scale, inverse=False):
    n = frequencies.numel()
    x = x.double()
    angle = positions.double()[..., None, None] * frequencies.double()
    c, s = angle.cos() * scale, angle.sin() * scale * (-1 if inverse else 1)
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    out, off = x.clone(), torch.zeros_like(x)
    p, q, e = a * c - b * s, b * c + a * s, 16 * W * (a.abs() + b.abs()) * abs(scale)
    for t, u, v in ((out, p, q), (off, e, e)):
        if interleaved:
            t[..., 0:2 * n:2], t[..., 1:2 * n:2] = u, v
        else:
            t[..., :n], t[..., n:2 * n] = u, v
    return out, off


def near(got, want, bound, name):
    u = U[got.dtype]
    limit = bound + u * (want.abs() + bound) + {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[got.dtype]
    worst = ((got.double() - want).abs() / limit).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times what it may be off"


def check(q, k, positions, frequencies, interleaved=False, scale=1.0):
    q, k = (t.detach().requires_grad_(True) if t is not None else None for t in (q, k))
    given = [t for t in (q, k) if t is not None]
    out = [t for t in rotary(q, k, positions, frequencies, interleaved=interleaved, scale=scale) if t is not None]
    grads = [torch.randn_like(t) for t in out]
    back = torch.autograd.grad(out, given, grads)
    for x, y, g, b in zip(given, out, grads, back):
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
        near(y.detach(), *exact(x.detach(), positions, frequencies, interleaved, scale), "forward")
        near(b, *exact(g, positions, frequencies, interleaved, scale, True), "backward")
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,kv,dim,part", [(1, 32, 8, 128, 128), (1, 1, 1, 2, 2), (7, 3, 1, 64, 64), (33, 12, 4, 80, 80), (50, 4, 4, 128, 96), (19, 5, 2, 72, 18),
                                                      (5, 2, 1, 13, 6), (300, 8, 2, 64, 32), (3, 40, 40, 256, 64), (2, 1, 1, 2048, 2048), (1000, 1, 1, 16, 16)])
def test_against_64_bits(tokens, heads, kv, dim, part, dtype, interleaved):
    g = torch.Generator().manual_seed(tokens + dim)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(dtype).to(DEV) for h in (heads, kv))
    f, _ = rotary_frequencies(part, device=DEV)
    check(q, k, torch.randint(0, 5000, (tokens,), generator=g).to(DEV), f, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(interleaved):
    """The angle of position 2^40 is as exact as that of 2: turns are counted in 64 bits."""
    f, _ = rotary_frequencies(64, 500000.0, device=DEV)
    p = torch.tensor([0, 1, -1, 131071, 1 << 20, (1 << 31) - 1, 1 << 31, -(1 << 33)], device=DEV)
    q = torch.randn(8, 4, 64, device=DEV)
    # (2^33 turns of the first pair in 64 bits leave 2^-19 of one: the reference itself is off by 2^33 2^-53)
    out = rotary(q, None, p, f, interleaved=interleaved)[0]
    want, bound = exact(q, p, f, interleaved, 1.0)
    near(out, want, bound + 4 * q.abs().max().item() * 2.0 ** (33 - 52), "far")
    assert torch.equal(out[0], q[0])


def test_positions_of_either_type_and_of_shared_dimensions():
    f, _ = rotary_frequencies(32, device=DEV)
    q, k = torch.randn(3, 20, 4, 32, device=DEV).bfloat16(), torch.randn(3, 20, 2, 32, device=DEV).bfloat16()
    p = torch.arange(20, device=DEV) + 7
    full = p.expand(3, 20)
    want = check(q, k, full, f)
    for pos in (p, p.int(), full.int().contiguous()):
        for a, b in zip(rotary(q, k, pos, f), want):
            assert torch.equal(a, b)
    one = rotary(q, k, torch.tensor(5, device=DEV), f)
    for a, b in zip(one, rotary(q, k, torch.full((3, 20), 5, device=DEV), f)):
        assert torch.equal(a, b)


def test_views():
    """Parts of one linear's output, heads in front of tokens, rows off 16-byte boundaries, the first positions of a cache."""
    f, _ = rotary_frequencies(64, device=DEV)
    p = torch.arange(90, device=DEV)
    qkv = torch.randn(90, 12, 64, device=DEV).bfloat16()
    q, k = qkv[:, :8], qkv[:, 8:10]
    want = check(q, k, p, f)
    odd = torch.nn.functional.pad(qkv, (1, 2))[..., 1:-2]
    for args in ((q.contiguous(), k.contiguous()), (q.transpose(0, 1).contiguous().transpose(0, 1), k), (odd[:, :8], odd[:, 8:10])):
        for a, b in zip(rotary(*args, p, f), want):
            assert torch.equal(a, b)
    cache = torch.randn(3, 40, 2, 64, device=DEV).half()
    part = cache[:, :17]
    p = torch.arange(17, device=DEV)
    assert torch.equal(rotary(part, None, p, f)[0], rotary(part.contiguous(), None, p, f)[0])
    strided = torch.arange(34, device=DEV)[::2]
    assert torch.equal(rotary(part, None, strided, f)[0], rotary(part, None, strided.contiguous(), f)[0])


@pytest.mark.parametrize("wanted", [(True, False), (False, True)])
def test_one_gradient_at_a_time(wanted):
    f, _ = rotary_frequencies(64, device=DEV)
    q, k = (torch.randn(9, h, 64, device=DEV).requires_grad_(w) for h, w in zip((4, 2), wanted))
    p = torch.arange(9, device=DEV)
    out = rotary(q, k, p, f)
    assert [t.requires_grad for t in out] == list(wanted)
    i = wanted.index(True)
    g = torch.randn_like(out[i])
    near(torch.autograd.grad(out[i], (q, k)[i], g)[0], *exact(g, p, f, False, 1.0, True), "gradient")


def test_gradient_of_one_output_alone():
    f, _ = rotary_frequencies(64, device=DEV)
    q, k = (torch.randn(9, h, 64, device=DEV).requires_grad_(True) for h in (4, 2))
    out = rotary(q, k, torch.arange(9, device=DEV), f)
    got = torch.autograd.grad(out[1].sum(), (q, k), allow_unused=True)
    assert got[0] is None and got[1] is not None


def test_many_tokens():
    f, _ = rotary_frequencies(64, device=DEV)
    q, k = (torch.randn(20011, h, 64, device=DEV).bfloat16() for h in (3, 1))
    check(q, k, torch.arange(20011, device=DEV), f, scale=1.25)


def test_more_than_2_32_bytes():
    """A block of tokens again and again: every one of its copies turns to the same bits, forward and backward."""
    copies, tokens, heads, dim = 280, 1000, 64, 128
    f, _ = rotary_frequencies(dim, device=DEV)
    block = torch.randn(tokens, heads, dim, device=DEV).bfloat16()
    q = block.repeat(copies, 1, 1).requires_grad_(True)
    assert q.numel() * 2 > 1 << 32
    out = rotary(q, None, torch.arange(tokens, device=DEV).repeat(copies), f)[0]
    (back,) = torch.autograd.grad(out, q, out.detach())
    first = check(block, None, torch.arange(tokens, device=DEV), f)[0].detach()
    for c in range(copies):
        rows = slice(c * tokens, (c + 1) * tokens)
        assert torch.equal(out[rows], first)
        assert torch.equal(back[rows], back[:tokens])


def test_another_stream_and_twice_backward():
    f, _ = rotary_frequencies(64, device=DEV)
    q, k = (torch.randn(500, h, 64, device=DEV).bfloat16().requires_grad_(True) for h in (4, 2))
    at = torch.arange(500, device=DEV)
    want = rotary(q, k, at, f)
    grads = torch.autograd.grad(want, (q, k), [t.detach() for t in want], retain_graph=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary(q, k, at, f)
        back = torch.autograd.grad(got, (q, k), [t.detach() for t in got])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*got, *back), (*want, *grads)))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, (q, k), [t.detach() for t in want]), grads))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(rotary(q, k, at, f), want))


def test_nothing_to_do():
    f, _ = rotary_frequencies(64, device=DEV)
    q = torch.zeros(0, 4, 64, device=DEV, requires_grad=True)
    out = rotary(q, None, torch.zeros(0, dtype=torch.int64, device=DEV), f)[0]
    assert out.shape == q.shape and torch.autograd.grad(out.sum(), q)[0].shape == q.shape


def test_module_keeps_its_frequencies_in_64_bits():
    m = RotaryEmbedding(128, 500000.0, dict(kind="yarn", factor=4.0, original=8192), rotary_dim=64, device=DEV).to(torch.bfloat16)
    assert m.frequencies.dtype == torch.float64 and m.frequencies.is_cuda
    q = torch.randn(10, 4, 128, device=DEV).bfloat16()
    p = torch.arange(10, device=DEV)
    f, s = rotary_frequencies(64, 500000.0, dict(kind="yarn", factor=4.0, original=8192), device=DEV)
    assert s == 0.1 * math.log(4.0) + 1.0
    assert torch.equal(m(q, None, p)[0], rotary(q, None, p, f, scale=s)[0])
    with pytest.raises(ValueError, match="128"):
        m(q[..., :64], None, p)


def test_graph_replays():
    f, _ = rotary_frequencies(64, device=DEV)
    q, k, p = torch.randn(70, 4, 64, device=DEV).bfloat16(), torch.randn(70, 2, 64, device=DEV).bfloat16(), torch.arange(70, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary(q, k, p, f)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rotary(q, k, p, f)
    for i in range(3):
        q.normal_()
        p.add_(100)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, rotary(q, k, p, f)):
            assert torch.equal(a, b), i


def test_refusals():
    f, _ = rotary_frequencies(64, device=DEV)
    q, k, p = torch.randn(6, 4, 64, device=DEV), torch.randn(6, 2, 64, device=DEV), torch.arange(6, device=DEV)
    for e, args, kw in ((TypeError, (q.double(), k.double(), p, f), {}), (TypeError, (q, k.half(), p, f), {}), (ValueError, (q, k[:5], p, f), {}), (ValueError, (q, k[..., :32], p, f), {}),
                        (ValueError, (q, k, p[:5], f), {}), (TypeError, (q, k, p.float(), f), {}), (TypeError, (q, k, p, f.float()), {}), (ValueError, (q[..., :32], k[..., :32], p, f), {}),
                        (ValueError, (q, k, p, f[:0]), {}), (ValueError, (q, k, p.cpu(), f), {}), (ValueError, (q, k, p, f.cpu()), {}), (ValueError, (q, k, p, f), dict(scale=math.inf)),
                        (ValueError, (q[0, 0], None, p, f), {}), (ValueError, (q, k, p, f.clone().requires_grad_(True)), {})):
        with pytest.raises(e):
            rotary(*args, **kw)
    leaf = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(rotary(leaf, None, p, f)[0].sum(), leaf, create_graph=True)
