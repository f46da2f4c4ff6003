"""AdamW against its formula in 64 bits.

Tolerances, u = 2^-24: moments are two products and a sum (3 u of the terms' magnitudes; the gradient times a factor one more); the
parameter moves by d = to m / (root r + eps): 8 u |d| more or less, and is rounded three times (3 u |p|), once more to its type.
Codes of 8-bit moments stand for one of the two neighbours of the value; neighbours are 2^-3 of the value apart at most, or
2^-9 / scale below the format's normal numbers."""
import copy

import pytest
import torch

from nanotron_amd.fp8 import DTypes, FP8Linear, FP8Parameter
from nanotron_amd.optim import AdamW, adamw_8bit_step, adamw_step, dequantize_moment, moments_8bit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def draw(n, dtype, gdtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    p = torch.randn(n, generator=g, device=DEV).mul_(0.05).to(dtype)
    grad = torch.randn(n, generator=g, device=DEV).mul_(1e-2).to(gdtype)
    m = torch.randn(n, generator=g, device=DEV).mul_(3e-3)
    v = torch.randn(n, generator=g, device=DEV).mul_(1e-2).square_()
    return p, grad, m, v


def exact(p, g, m, v, step, scale=1.0, lr=0, betas=0, eps=0, weight_decay=0):
    p, g, m, v = p.double(), g.double() * scale, m.double(), v.double()
    m2 = betas[0] * m + (1 - betas[0]) * g
    v2 = betas[1] * v + (1 - betas[1]) * g * g
    d = lr / (1 - betas[0] ** step) * m2 / (v2.sqrt() / (1 - betas[1] ** step) ** 0.5 + eps)
    em = 5 * U32 * (betas[0] * m.abs() + (1 - betas[0]) * g.abs())
    ev = 8 * U32 * v2
    # the error of m reaches the step as a share of it, also where the sum of its terms is nearly nothing
    ed = 12 * U32 * d.abs() + lr / (1 - betas[0] ** step) * em / (v2.sqrt() / (1 - betas[1] ** step) ** 0.5 + eps)
    q = p * (1 - lr * weight_decay) - d
    return (q, m2, v2), (3 * U32 * (p.abs() + d.abs()) + ed, em, ev)


def near(got, want, bound, name):
    u = U[got.dtype]
    limit = bound + u * (want.abs() + bound) + {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[got.dtype]
    worst = ((got.double() - want).abs() / limit).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times what it may be off"


TYPES = [(torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.bfloat16, None),
         (torch.float16, torch.float16, torch.float32), (torch.float32, torch.float16, torch.float16)]
LENGTHS = [1, 2, 3, 5, 255, 256, 257, 1023, 4095, 4096, 4097, 70001]


@pytest.mark.parametrize("dtype,gdtype,cdtype", TYPES)
def test_step_32(dtype, gdtype, cdtype):
    data = [draw(n, dtype, gdtype, i) for i, n in enumerate(LENGTHS + [0])]
    before = [[t.clone() for t in d] for d in data]
    copies = None if cdtype is None else [torch.zeros(d[0].shape, dtype=cdtype, device=DEV) for d in data]
    clip = torch.full((1,), 0.5, device=DEV)
    adamw_step(*[list(c) for c in zip(*data)], step=7, grad_scale=clip, copies=copies, **HYPER)
    for i, (d, old) in enumerate(zip(data, before)):
        want, bound = exact(*old, step=7, scale=0.5, **HYPER)
        for k, name in ((0, "param"), (2, "exp_avg"), (3, "exp_avg_sq")):
            near(d[k], want[(0, 0, 1, 2)[k]], bound[(0, 0, 1, 2)[k]], f"{name} of {d[0].numel()}")
        assert torch.equal(d[1], old[1])
        if copies is not None:
            near(copies[i], want[0], bound[0], "copy")


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_unaligned_tensors(offset):
    """Views that begin on any element, each with its own neighbours, which stay as they are."""
    n = 5003
    for dtype, gdtype in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)):
        p, g, m, v = draw(n + 8, dtype, gdtype, offset)
        old = [t.clone() for t in (p, g, m, v)]
        at = slice(offset, offset + n)
        adamw_step([p[at]], [g[at]], [m[at]], [v[at]], step=3, **HYPER)
        want, bound = exact(*[t[at] for t in old], step=3, **HYPER)
        near(p[at], want[0], bound[0], "param")
        near(m[at], want[1], bound[1], "exp_avg")
        for t, o in zip((p, m, v), (old[0], old[2], old[3])):
            assert torch.equal(t[:offset], o[:offset]) and torch.equal(t[offset + n:], o[offset + n:])


def packed(n, m, r):
    """Codes and scales whose values are what a first 8-bit step made of m and r from zero moments (betas of 0: g itself)."""
    mc, ms, rc, rs = moments_8bit(torch.empty(n, device=DEV))
    adamw_8bit_step([torch.zeros(n, device=DEV)], [r], [mc], [ms], [rc], [rs], lr=0.0, betas=(0.0, 0.0), step=1, seed=5)
    mc2, ms2, _, _ = moments_8bit(torch.empty(n, device=DEV))
    spare = moments_8bit(torch.empty(n, device=DEV))
    adamw_8bit_step([torch.zeros(n, device=DEV)], [m], [mc2], [ms2], [spare[2]], [spare[3]], lr=0.0, betas=(0.0, 0.0), step=1, seed=6)
    return mc2, ms2, rc, rs


def check_codes(codes, scales, want, bound, root):
    """Codes stand for a neighbour of the value; the block's scale brings its largest magnitude into (224, 448]."""
    n = want.numel()
    got = dequantize_moment(codes, scales).double()
    per = scales.double().repeat_interleave(256)[:n]
    gap = torch.maximum(want.abs() * 2.0 ** -3, 2.0 ** -9 / per)
    assert ((got - want).abs() <= gap + bound).all()
    pad = torch.nn.functional.pad(want.abs(), (0, -n % 256)).view(-1, 256).amax(-1)
    top = pad * scales.double()
    some = pad > 0
    assert (scales[~some] == 1).all()
    assert (top[some] > 224 * (1 - 1e-5)).all() and (top[some] <= 448 * (1 + 1e-5)).all()
    assert (torch.frexp(scales)[0] == 0.5).all()
    if root:
        assert (got[want > 0] > 0).all() and (codes.view(torch.int8) >= 0).all()


@pytest.mark.parametrize("dtype,gdtype,cdtype", TYPES)
def test_step_8(dtype, gdtype, cdtype):
    data, old, lists = [], [], []
    for i, n in enumerate(LENGTHS):
        p, g, m, v = draw(n, dtype, gdtype, 100 + i)
        st = packed(n, m, v.sqrt())
        data.append((p, g, *st))
        old.append((p.clone(), g.clone(), dequantize_moment(st[0], st[1]), dequantize_moment(st[2], st[3])))
    copies = None if cdtype is None else [torch.zeros(d[0].shape, dtype=cdtype, device=DEV) for d in data]
    lists = [list(c) for c in zip(*data)]
    adamw_8bit_step(*lists, step=9, seed=1234, copies=copies, **HYPER)
    for i, (d, o) in enumerate(zip(data, old)):
        want, bound = exact(o[0], o[1], o[2], o[3].double() ** 2, step=9, **HYPER)
        near(d[0], want[0], bound[0], f"param of {d[0].numel()}")
        check_codes(d[2], d[3], want[1], bound[1], False)
        check_codes(d[4], d[5], want[2].sqrt(), 8 * U32 * want[2].sqrt(), True)
        if copies is not None:
            near(copies[i], want[0], bound[0], "copy")


def test_rounding_is_unbiased_and_seeded():
    n = 1 << 18
    value = torch.full((n,), 0.7371, device=DEV)
    value[::256] = 1.0   # the blocks' largest
    out = []
    for seed in (1, 1, 2):
        mc, ms, rc, rs = moments_8bit(value)
        adamw_8bit_step([torch.zeros(n, device=DEV)], [value], [mc], [ms], [rc], [rs], lr=0.0, betas=(0.0, 0.0), step=1, seed=seed)
        out.append(mc)
        for codes, scales in ((mc, ms), (rc, rs)):
            got = dequantize_moment(codes, scales)
            pick = torch.ones(n, dtype=torch.bool, device=DEV)
            pick[::256] = False
            assert got[pick].unique().numel() == 2   # the two neighbours
            # two neighbours 1/16 apart: a standard error of at most 1/32 / sqrt(n); six of them
            assert abs(got[pick].double().mean().item() - 0.7371) < 6 / 32 / n ** 0.5
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])


def test_a_falling_root_falls():
    """beta2 = 0.999 without gradient: the root falls by 0.05 % a step, far less than a step of its format."""
    n = 1 << 14
    p = torch.zeros(n, device=DEV)
    g = torch.rand(n, device=DEV) + 0.5
    mc, ms, rc, rs = moments_8bit(p)
    adamw_8bit_step([p], [g], [mc], [ms], [rc], [rs], lr=0.0, betas=(0.0, 0.0), step=1, seed=0)
    start = dequantize_moment(rc, rs).double().square().mean().item()
    for t in range(200):
        adamw_8bit_step([p], [torch.zeros_like(g)], [mc], [ms], [rc], [rs], lr=0.0, betas=(0.9, 0.999), step=2 + t, seed=100 + t)
    end = dequantize_moment(rc, rs).double().square().mean().item()
    # A step leaves 0.999 of r^2, and rounding without bias adds its variance: at most 0.0005 r times a gap of r / 8.  Over 200
    # steps 0.8187 to 0.829, give or take six standard errors of 2^14 elements (0.13 / 2^7 each)
    assert 0.8187 - 0.0061 < end / start < 0.829 + 0.0061


def test_specials():
    p, g, m, v = draw(1024, torch.float32, torch.float32)
    g[3], g[700] = float("nan"), float("inf")
    q, m2, v2 = p.clone(), m.clone(), v.clone()
    adamw_step([q], [g], [m2], [v2], step=2, **HYPER)
    bad = torch.zeros(1024, dtype=torch.bool, device=DEV)
    bad[3] = bad[700] = True
    assert torch.equal(q.isnan(), bad) and torch.equal(m2.isfinite(), ~bad)
    st = packed(1024, m, v.sqrt())
    q = p.clone()
    adamw_8bit_step([q], [g], [st[0]], [st[1]], [st[2]], [st[3]], step=2, seed=3, **HYPER)
    assert torch.equal(q.isnan(), bad)
    assert torch.equal(dequantize_moment(st[0], st[1]).isnan(), bad) and torch.equal(dequantize_moment(st[2], st[3]).isnan(), bad)
    # zeros stay zeros with a scale of one; tiny values keep a finite scale
    z = torch.zeros(512, device=DEV)
    z[300] = 1e-42
    st = moments_8bit(z)
    adamw_8bit_step([torch.zeros_like(z)], [z], [st[0]], [st[1]], [st[2]], [st[3]], lr=0.0, betas=(0.0, 0.0), step=1, seed=3)
    assert st[1][0] == 1 and st[1].isfinite().all() and st[3].isfinite().all() and (st[0][:256] == 0).all()


def test_many_tensors_in_one_call():
    """More tensors than one launch takes, types mixed."""
    data = [draw(1 + 37 * i, (torch.float32, torch.bfloat16)[i % 2], (torch.float32, torch.bfloat16)[i % 2], i) for i in range(130)]
    old = [[t.clone() for t in d] for d in data]
    adamw_step(*[list(c) for c in zip(*data)], step=5, **HYPER)
    for d, o in zip(data, old):
        want, bound = exact(*o, step=5, **HYPER)
        near(d[0], want[0], bound[0], "param")


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_the_memory_side_cache(bits):
    """Steps that move over 256 MB take another path to memory: 24 million elements beside an odd few."""
    hyper = dict(HYPER, step=4)
    big = 24_000_003
    for dtype, gdtype in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)):
        data = [draw(n, dtype, gdtype, n) for n in (big, 77)]
        if bits == 32:
            old = [[t.clone() for t in d] for d in data]
            adamw_step(*[list(c) for c in zip(*data)], **hyper)
            for d, o in zip(data, old):
                want, bound = exact(*o, **hyper)
                for k, name in ((0, "param"), (2, "exp_avg"), (3, "exp_avg_sq")):
                    near(d[k], want[(0, 0, 1, 2)[k]], bound[(0, 0, 1, 2)[k]], name)
        else:
            full = [(p, g, *packed(p.numel(), m, v.sqrt())) for p, g, m, v in data]
            old = [(p.clone(), g, dequantize_moment(a, b), dequantize_moment(c, e)) for p, g, a, b, c, e in full]
            adamw_8bit_step(*[list(c) for c in zip(*full)], seed=8, **hyper)
            for d, o in zip(full, old):
                want, bound = exact(o[0], o[1], o[2], o[3].double() ** 2, **hyper)
                near(d[0], want[0], bound[0], "param")
                check_codes(d[2], d[3], want[1], bound[1], False)
                check_codes(d[4], d[5], want[2].sqrt(), 8 * U32 * want[2].sqrt(), True)


def test_optimizer_follows_torch():
    """32-bit moments: the optimizer beside torch.optim.AdamW in 64 bits, over 20 steps; 8-bit moments stay near."""
    torch.manual_seed(0)
    shapes = [(64, 33), (257,), (1,), (128, 128)]
    start = [torch.randn(s) * 0.1 for s in shapes]
    ours = [torch.nn.Parameter(t.to(DEV)) for t in start]
    small = [torch.nn.Parameter(t.to(DEV)) for t in start]
    ref = [torch.nn.Parameter(t.double().to(DEV)) for t in start]
    a, b, c = AdamW(ours, **HYPER), torch.optim.AdamW(ref, **HYPER), AdamW(small, state_bits=8, **HYPER)
    for k in range(20):
        for x, y, z in zip(ours, ref, small):
            g = torch.randn(x.shape, device=DEV) * (1 + torch.randn(x.shape, device=DEV).abs())
            x.grad, y.grad, z.grad = g, g.double(), g.clone()
        for o in (a, b, c):
            o.step()
    moved = sum((y.detach() - s.to(DEV).double()).square().sum() for y, s in zip(ref, start)).sqrt().item()
    off = sum((x.detach().double() - y.detach()).square().sum() for x, y in zip(ours, ref)).sqrt().item()
    off8 = sum((x.detach().double() - y.detach()).square().sum() for x, y in zip(small, ref)).sqrt().item()
    # 20 steps of a rounding each; codes with 1/16 steps on both moments leave a step off by at most 1/8
    assert off < 1e-5 * moved and off8 < 0.125 * moved


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    torch.manual_seed(1)
    p = [torch.nn.Parameter(torch.randn(300, device=DEV).bfloat16()), torch.nn.Parameter(torch.randn(40, 9, device=DEV))]
    o = AdamW(p, state_bits=bits, **HYPER)
    for q in p:
        q.grad = torch.randn_like(q)
    o.step()
    q = [torch.nn.Parameter(x.detach().clone()) for x in p]
    r = AdamW(q, state_bits=bits, **HYPER)
    r.load_state_dict(copy.deepcopy(o.state_dict()))
    for x, y in zip(p, q):
        for k, v in o.state[x].items():
            w = r.state[y][k]
            assert (torch.equal(v, w) and v.dtype == w.dtype) if isinstance(v, torch.Tensor) else v == w
        x.grad = torch.randn_like(x)
        y.grad = x.grad.clone()
    o.step()
    r.step()
    assert all(torch.equal(x, y) for x, y in zip(p, q))


def test_fp8_linear_masters_and_copies():
    """What an FP8Linear's weight accumulates (main_grad beside a 16-bit master, grad beside an fp32 one) steps its master."""
    for dtype in (torch.bfloat16, torch.float32):
        lin = FP8Linear(256, 128, bias=True, device=DEV, dtype=dtype, out_dtype=torch.bfloat16)
        lin.weight = FP8Parameter((0.02 * torch.randn(128, 256, device=DEV)).to(dtype), DTypes.FP8E4M3)
        o = AdamW(lin.parameters(), **HYPER)
        before = lin.weight.as_subclass(torch.Tensor).detach().clone()
        lin(torch.randn(64, 256, device=DEV, dtype=torch.bfloat16)).float().square().mean().backward()
        grad = lin.weight.grad if lin.weight.grad is not None else lin.weight.main_grad
        o.step()
        zero = torch.zeros(before.shape, device=DEV)
        want, bound = exact(before, grad.as_subclass(torch.Tensor), zero, zero, step=1, **HYPER)
        near(lin.weight.as_subclass(torch.Tensor).detach(), want[0], bound[0], "weight")
    master = torch.nn.Parameter(torch.randn(1000, device=DEV))
    model = torch.zeros(1000, device=DEV, dtype=torch.bfloat16)
    o = AdamW([dict(params=[master], copies=[model])], **HYPER)
    master.grad = torch.randn(1000, device=DEV)
    o.step(grad_scale=torch.ones(1, device=DEV))
    assert torch.equal(model, master.detach().bfloat16())
    assert o.state_dict()["param_groups"][0]["copies"] is None


def test_refusals():
    p, g, m, v = draw(64, torch.float32, torch.float32)
    good = dict(lr=1e-3, step=1)
    for args, error in ((([p], [g], [m], []), ValueError), (([p], [g[:63]], [m], [v]), ValueError), (([p], [g], [m.half()], [v]), TypeError),
                        (([p], [g.cpu()], [m], [v]), ValueError), (([p.double()], [g], [m], [v]), TypeError),
                        (([torch.zeros(64, 2, device=DEV)[:, 0]], [g], [m], [v]), ValueError)):
        with pytest.raises(error):
            adamw_step(*args, **good)
    with pytest.raises(ValueError, match="step"):
        adamw_step([p], [g], [m], [v], lr=1e-3, step=0)
    with pytest.raises(ValueError, match="betas"):
        adamw_step([p], [g], [m], [v], lr=1e-3, step=1, betas=(0.9, 1.0))
    with pytest.raises(TypeError, match="grad_scale"):
        adamw_step([p], [g], [m], [v], grad_scale=torch.ones(2, device=DEV), **good)
    with pytest.raises(RuntimeError, match="overlap"):
        adamw_step([p], [p], [m], [v], **good)
    with pytest.raises(ValueError, match="scales"):
        adamw_8bit_step([p], [g], [m.byte()], [torch.ones(2, device=DEV)], [v.byte()], [torch.ones(1, device=DEV)], seed=0, **good)


def test_autograd_sees_new_copies():
    """A product that saved a 16-bit copy cannot be differentiated through once a step has changed it."""
    master = torch.nn.Parameter(torch.randn(8, 8, device=DEV))
    model = master.detach().bfloat16().requires_grad_(True)
    out = (torch.ones(2, 8, device=DEV, dtype=torch.bfloat16, requires_grad=True) * model[:2]).sum()
    master.grad = torch.ones_like(master)
    AdamW([dict(params=[master], copies=[model])], **HYPER).step()
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward()


def test_a_refused_step_is_not_counted():
    p = torch.nn.Parameter(torch.randn(8, 8, device=DEV))
    o = AdamW([p], **HYPER)
    p.grad = torch.ones_like(p)
    with pytest.raises(TypeError, match="grad_scale"):
        o.step(grad_scale=torch.ones(2, device=DEV))
    assert o.state[p]["step"] == 0
    o.step()
    assert o.state[p]["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays(bits):
    """A captured step, replayed with new gradients and other work in between, is the step launched from Python."""
    tensors = [draw(n, torch.float32, torch.bfloat16, seed=n) for n in (70001, 256, 5)]
    params, grads, ms, vs = ([t[i].clone() for t in tensors] for i in range(4))
    factor = torch.full((1,), 0.5, device=DEV)
    state = [moments_8bit(p) for p in params]

    def step(params, ms, vs, state):
        if bits == 32:
            adamw_step(params, grads, ms, vs, step=3, grad_scale=factor, **HYPER)
        else:
            m, s, r, t = zip(*state)
            adamw_8bit_step(params, grads, m, s, r, t, step=3, seed=11, grad_scale=factor, **HYPER)

    def clones():
        return [p.clone() for p in params], [m.clone() for m in ms], [v.clone() for v in vs], [tuple(t.clone() for t in s) for s in state]

    mine = clones()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*clones())
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(params, ms, vs, state)
    for k in range(4):
        for g in grads:
            g.copy_(torch.randn(g.shape, device=DEV) * 10.0 ** -k)
        step(*mine)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mine[0], params)), k
        assert all(torch.equal(a, b) for s, t in zip(mine[3], state) for a, b in zip(s, t)), k


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_beyond_32_bits(bits):
    """A tensor of more than 2^32 bytes, which a launch takes as several: the elements where one ends and the last ones."""
    n = (1 << 31) + 1027
    p, g = (torch.randn(n, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    parts = [slice(0, 5000), slice((1 << 30) - 2560, (1 << 30) + 2560), slice((1 << 31) - 2560, n)]
    before = [p[s].clone() for s in parts]
    if bits == 32:
        m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
        adamw_step([p], [g], [m], [v], step=1, **HYPER)
    else:
        state = moments_8bit(p)
        adamw_8bit_step([p], [g], *([t] for t in state), step=1, seed=5, **HYPER)
    for s, old in zip(parts, before):
        zero = torch.zeros(old.shape, device=DEV)
        want, bound = exact(old, g[s], zero, zero, step=1, **HYPER)
        near(p[s], want[0], bound[0], "parameter")
        if bits == 32:
            near(m[s], want[1], bound[1], "first moment")
            near(v[s], want[2], bound[2], "second moment")
        else:
            # a code is a neighbour of its value: an eighth of it off at most, or the distance of the smallest codes
            blocks = slice(s.start // 256, -(-s.stop // 256))
            for code, scale, value in ((state[0], state[1], want[1]), (state[2], state[3], want[2].sqrt())):
                got = dequantize_moment(code[blocks.start * 256:s.stop], scale[blocks])[s.start - blocks.start * 256:]
                each = scale[blocks].repeat_interleave(256)[s.start - blocks.start * 256:][:got.numel()].double()
                assert ((got.double() - value).abs() <= value.abs() / 8 + 2.0 ** -9 / each).all()
    del p, g
    torch.cuda.empty_cache()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bad_gradient_costs_its_own_elements(dtype, value):
    """8-bit moments: one step with gradients that are not finite, three with finite ones.  Only those elements are lost: their
    neighbours' codes and scales, and the parameters that the next steps make of them, are as if the block held nothing else."""
    n, where = 1500, [0, 5, 255, 700, 702, 1499]
    p, g, m, v = draw(n, dtype, torch.float32, 3)
    st = packed(n, m, v.sqrt())
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[where] = True
    bad[256:512] = True      # a block with nothing else in it
    for step in range(2, 6):
        grad = torch.where(bad, value, g) if step == 2 else g * (step - 3.5)
        old = (p.clone(), dequantize_moment(st[0], st[1]), dequantize_moment(st[2], st[3]))
        adamw_8bit_step([p], [grad], *([t] for t in st), step=step, seed=step, **HYPER)
        assert torch.equal(p.isnan(), bad), step
        want, bound = exact(old[0], grad, old[1], old[2].double() ** 2, step=step, **HYPER)
        near(p[~bad], want[0][~bad], bound[0][~bad], f"param in step {step}")
        for codes, scales, value_of, off, root in ((st[0], st[1], want[1], bound[1], False), (st[2], st[3], want[2].sqrt(), 8 * U32 * want[2].sqrt(), True)):
            assert torch.equal(dequantize_moment(codes, scales).isnan(), bad), step
            clean = [torch.where(bad, torch.zeros_like(t), t) for t in (codes, value_of, off)]
            check_codes(clean[0], scales, clean[1], clean[2], root)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_call_has_stepped_nothing(bits):
    """Of tensors of two sets of types the second set is refused: the first one stays as it was, too."""
    data = [draw(1000, dtype, dtype, i) for i, dtype in enumerate((torch.bfloat16, torch.float32))]
    params, grads = [d[0] for d in data], [data[0][1], data[1][0]]      # (the second gradient is the parameter itself)
    state = [moments_8bit(p) for p in params] if bits == 8 else [(d[2], d[3]) for d in data]
    held = [*params, *state[0], *state[1]]
    before, versions = [t.clone() for t in held], [t._version for t in held]
    with pytest.raises(RuntimeError, match="overlap"):
        (adamw_step if bits == 32 else adamw_8bit_step)(params, grads, *map(list, zip(*state)), step=1, **HYPER, **({} if bits == 32 else dict(seed=2)))
    assert all(torch.equal(a, b) for a, b in zip(held, before)) and versions == [t._version for t in held]
    p = [torch.nn.Parameter(d[0].clone()) for d in data]
    o = AdamW(p, state_bits=bits, **HYPER)
    p[0].grad, p[1].grad = data[0][1], p[1].data
    before = [q.detach().clone() for q in p]
    with pytest.raises(RuntimeError, match="overlap"):
        o.step()
    assert all(torch.equal(q.detach(), b) for q, b in zip(p, before)) and o.state[p[0]]["step"] == 0


def test_dither_of_a_tensor_beyond_a_launch():
    """Codes are rounded by the hash of the element's index in its tensor, also where a launch takes the tensor in parts (of
    2^30 elements): the hash in Python's integers says which of the two neighbours of 0.7371 every element gets."""
    n, seed = (1 << 30) + 5003, 77
    p, g = torch.zeros(n, device=DEV, dtype=torch.bfloat16), torch.full((n,), 0.7371, device=DEV, dtype=torch.bfloat16)
    g[::256] = 1.0      # the blocks' largest: a scale of 256
    state = moments_8bit(p)
    adamw_8bit_step([p], [g], *([t] for t in state), lr=0.0, betas=(0.0, 0.0), step=1, seed=seed)
    assert (state[1] == 256).all()

    def code(i, value):
        mask = 0xFFFFFFFF
        x = ((i >> 1) * 0x9E3779B1 + seed * 0xBB67AE85) & mask
        x = (x ^ x >> 15) * 0x6A09E667 & mask
        x = (x ^ x >> 13) * 0x3C6EF373 & mask
        x ^= x >> 16
        bits = torch.tensor(value * 256).view(torch.int32).item()
        return ((bits + ((x >> 16 if i & 1 else x & 0xFFFF) << 4)) >> 20) - 960

    value = g[1].item()
    for first in (0, (1 << 30) - 512, 1 << 30, n - 512):
        want = [code(i, 1.0 if i % 256 == 0 else value) for i in range(first, first + 512)]
        assert len(set(want)) == 3 and state[0][first:first + 512].tolist() == want, first
    del p, g, state
    torch.cuda.empty_cache()


def test_goes_on_from_a_torch_optimizer():
    """A state dict of torch.optim.AdamW: the moments (fp32, whatever the parameters' type) and counts of steps are taken over, and
    the next step is that of the formula."""
    start = [draw(n, dtype, dtype, n)[0] for n, dtype in ((300, torch.float32), (700, torch.bfloat16))]
    ref = [torch.nn.Parameter(t.clone()) for t in start]
    theirs = torch.optim.AdamW(ref, **HYPER)
    for k in range(3):
        for i, p in enumerate(ref):
            p.grad = draw(p.numel(), p.dtype, p.dtype, 10 * k + i)[1]
        theirs.step()
    own = [torch.nn.Parameter(p.detach().clone()) for p in ref]
    ours = AdamW(own, lr=1.0)
    ours.load_state_dict(theirs.state_dict())
    for p, q in zip(own, ref):
        assert ours.state[p]["step"] == 3 and type(ours.state[p]["step"]) is int
        m, v = (theirs.state[q][k] for k in ("exp_avg", "exp_avg_sq"))
        p.grad = draw(p.numel(), p.dtype, p.dtype, 99)[1]
        want, bound = exact(p.detach(), p.grad, m, v, step=4, **HYPER)
        q.want = want[0], bound[0]
    ours.step()
    for p, q in zip(own, ref):
        near(p.detach(), *q.want, "param")
        assert ours.state[p]["step"] == 4
