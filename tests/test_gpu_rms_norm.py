"""The norms around a block against their formulas in 64 bits.

Tolerances, with w = 2^-24: a sum of squares over up to 2^14 elements, a tree of at most 32 additions behind one another (mean, root and quotient 6
more), leaves 1 / rms off by 20 w; p by 24 w |p|, the sum of residual and gate p by 3 w of its terms more.  h is compared before and after its own rounding, and
y with the exact norm of the h that came back, so that no rounding counts twice.  The backward formulas likewise start from that h; sums of products are
bounded by the sums of magnitudes, in the order of the terms below, and sums over rows by (rows / 8 + 64) w of theirs."""
import pytest
import torch

from nanotron_amd.nn import RMSNorm, residual_rms_norm, rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W = 2.0 ** -24
EPS = 1e-6


def near(got, want, bound, name):
    u = U[got.dtype]
    limit = bound + u * (want.abs() + bound) + {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[got.dtype]
    off = (got.double() - want).abs()
    worst = (off / limit.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times what it may be off"


def inputs(rows, cols, dtype, rdtype, wdtype, post, gate, seed=0):
    g = torch.Generator().manual_seed(seed + rows + cols)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g) * std + mean

    s = dict(x=normal(rows, cols).to(dtype), residual=normal(rows, cols, std=2.0).to(rdtype), weight=normal(cols, std=0.2, mean=1.0).to(wdtype), post_weight=None, gate=None)
    if post:
        s["post_weight"] = normal(cols, std=0.2, mean=0.7).to(wdtype)
    if gate == "channel":
        s["gate"] = normal(cols, std=0.3, mean=0.3).to(wdtype)
    if gate == "element":
        s["gate"] = torch.sigmoid(normal(rows, cols)).to(dtype)
    s = {k: None if v is None else v.to(DEV) for k, v in s.items()}
    return s, normal(rows, cols).to(dtype).to(DEV), normal(rows, cols).to(rdtype).to(DEV)


def exact(s, h_got, dy, dh_out, scale):
    """{name: (value, what it may be off by)}; y and the gradients from the h that came back."""
    f = {k: None if v is None else v.detach().double() for k, v in s.items()}
    x, r, w, pw, gate = f["x"], f["residual"], f["weight"], f["post_weight"], f["gate"]
    one = torch.ones((), dtype=torch.float64, device=x.device)
    w = one if w is None else w
    first = (x.square().mean(-1, keepdim=True) + EPS).rsqrt() if pw is not None else one
    u = x * first
    p = u * pw if pw is not None else u
    e_p = 24 * W * p.abs() if pw is not None else 0 * p
    g = one if gate is None else gate
    h = scale * r + g * p
    out = {"h": (h, g.abs() * e_p + 3 * W * ((scale * r).abs() + (g * p).abs()))}
    hg = h_got.detach().double()
    second = (hg.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = hg * second
    out["y"] = (n * w, 24 * W * (n * w).abs())
    dy, do = dy.double(), dh_out.double()
    a = dy * w
    m = (a * n).mean(-1, keepdim=True)
    mm = (a * n).abs().mean(-1, keepdim=True)
    dh = do + second * (a - n * m)
    e_dh = W * (4 * do.abs() + second * (26 * a.abs() + n.abs() * (90 * mm)) + 4 * dh.abs())
    rows = (x.shape[0] / 8 + 72) * W
    out["weight"] = ((dy * n).sum(0), (rows + 24 * W) * (dy * n).abs().sum(0))
    out["residual"] = (scale * dh, abs(scale) * (e_dh + W * dh.abs()))
    if gate is not None:
        t, e = dh * p, e_dh * p.abs() + dh.abs() * e_p + 2 * W * (dh * p).abs()
        out["gate"] = (t, e) if gate.dim() == 2 else (t.sum(0), e.sum(0) + rows * t.abs().sum(0))
    dp, e_dp = dh * g, g.abs() * e_dh + W * (dh * g).abs()
    if pw is not None:
        out["post_weight"] = ((dp * u).sum(0), (e_dp * u.abs() + (24 * W + rows) * (dp * u).abs()).sum(0))
        q, e_q = dp * pw, e_dp * pw.abs() + W * (dp * pw).abs()
        mq, eq = (q * u).mean(-1, keepdim=True), (e_q * u.abs() + 60 * W * (q * u).abs()).mean(-1, keepdim=True)
        dx = first * (q - u * mq)
        out["x"] = (dx, first * (e_q + 26 * W * q.abs() + u.abs() * (eq + 50 * W * mq.abs())) + 4 * W * dx.abs())
    else:
        out["x"] = (dp, e_dp)
    return out


def check(s, dy, dh, scale=1.0):
    s = {k: None if v is None else v.detach().requires_grad_(True) for k, v in s.items()}
    y, h = residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], residual_scale=scale, eps=EPS)
    names = [k for k, v in s.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad((y, h), [s[k] for k in names], (dy, dh))))
    want = exact(s, h, dy, dh, scale)
    assert y.dtype == s["x"].dtype and h.dtype == s["residual"].dtype
    for k, got in (("h", h.detach()), ("y", y.detach()), *grads.items()):
        if k in s:
            assert got.shape == s[k].shape and got.dtype == s[k].dtype, k
        near(got, *want[k], k)
    with torch.no_grad():
        again = residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], residual_scale=scale, eps=EPS)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)
    return y, h, grads


TYPES = [(torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32, torch.float32),
         (torch.float16, torch.float16, torch.float32), (torch.float16, torch.float32, torch.float16)]
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 513), (17, 512), (33, 1000), (7, 1037), (130, 2048), (1021, 2049), (300, 4096), (5, 4097), (40, 8192)]


@pytest.mark.parametrize("post,gate", [(False, None), (True, "channel"), (True, "element")])
@pytest.mark.parametrize("dtype,rdtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_against_64_bits(rows, cols, dtype, rdtype, wdtype, post, gate):
    check(*inputs(rows, cols, dtype, rdtype, wdtype, post, gate), scale=0.5 if post else 1.0)


@pytest.mark.parametrize("post,gate", [(True, None), (False, "channel"), (False, "element")])
def test_every_part_alone(post, gate):
    for dtype, rdtype, wdtype in TYPES:
        check(*inputs(29, 640, dtype, rdtype, wdtype, post, gate), scale=-1.5)


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 16384), (torch.bfloat16, 12001), (torch.float32, 8192), (torch.float32, 5000)])
def test_widest_rows(dtype, cols):
    check(*inputs(6, cols, dtype, torch.float32, torch.float32, True, "channel"))


def test_many_rows():
    s, dy, dh = inputs(20011, 192, torch.bfloat16, torch.bfloat16, torch.float32, True, "channel")
    first = check(s, dy, dh)[2]
    again = check(s, dy, dh)[2]
    assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (37, 63), (300, 1037), (5, 8192)])
def test_norm_alone(rows, cols, dtype, wdtype):
    s, dy, _ = inputs(rows, cols, dtype, dtype, wdtype, False, None)
    x, w = s["x"].requires_grad_(True), s["weight"].requires_grad_(True)
    y = rms_norm(x, w, EPS)
    got = dict(zip(("x", "weight"), torch.autograd.grad(y, (x, w), dy)))
    # the same with h = x: a residual of zeros
    want = exact({**s, "residual": torch.zeros_like(x)}, x, dy, torch.zeros_like(x), 1.0)
    near(y.detach(), *want["y"], "y")
    near(got["x"], *want["residual"], "x")
    near(got["weight"], *want["weight"], "weight")
    with torch.no_grad():
        assert torch.equal(rms_norm(x, w, EPS), y)


def test_without_weight():
    s, dy, dh = inputs(21, 320, torch.bfloat16, torch.float32, torch.float32, True, None)
    check({**s, "weight": None}, dy, dh)
    x = s["x"].requires_grad_(True)
    assert torch.equal(rms_norm(x, None, EPS), rms_norm(x, torch.ones(320, device=DEV), EPS))


@pytest.mark.parametrize("which", ["x", "residual", "weight", "post_weight", "gate"])
def test_one_gradient_at_a_time(which):
    for gate in ("channel", "element"):
        s, dy, dh = inputs(50, 300, torch.bfloat16, torch.bfloat16, torch.bfloat16, True, gate)
        every = check(s, dy, dh)[2]
        leaf = s[which].requires_grad_(True)
        y, h = residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], eps=EPS)
        assert torch.equal(torch.autograd.grad((y, h), leaf, (dy, dh))[0], every[which])


@pytest.mark.parametrize("post,gate", [(False, None), (True, "channel")])
def test_one_output_alone(post, gate):
    s, dy, dh = inputs(19, 260, torch.bfloat16, torch.bfloat16, torch.float32, post, gate)
    s = {k: None if v is None else v.requires_grad_(True) for k, v in s.items()}
    names = [k for k, v in s.items() if v is not None]
    zero = torch.zeros_like(dy)
    for pick, pair in ((0, (dy, zero)), (1, (zero, dh))):
        out = residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], eps=EPS)
        got = torch.autograd.grad(out[pick], [s[k] for k in names], pair[pick])
        want = exact(s, out[1], *pair, 1.0)
        for k, g in zip(names, got):
            near(g, *want[k], k)


def test_gradients_do_not_share_what_a_caller_changes():
    """x and the residual may get one tensor: what is added to one later is added beside it."""
    s, dy, dh = inputs(8, 64, torch.bfloat16, torch.bfloat16, torch.float32, False, None)
    x, r = s["x"].requires_grad_(True), s["residual"].requires_grad_(True)
    for _ in range(2):
        torch.autograd.backward(residual_rms_norm(x, r, s["weight"], eps=EPS), (dy, dh))
    x2, r2 = (t.detach().clone().requires_grad_(True) for t in (x, r))
    torch.autograd.backward(residual_rms_norm(x2, r2, s["weight"], eps=EPS), (dy, dh))
    assert torch.equal(x.grad, 2 * x2.grad) and torch.equal(r.grad, 2 * r2.grad)
    # the same tensor as both
    t = x.detach().clone().requires_grad_(True)
    y, h = residual_rms_norm(t, t, s["weight"], eps=EPS)
    g = torch.autograd.grad((y, h), t, (dy, dh))[0]
    a, b = (x.detach().clone().requires_grad_(True) for _ in range(2))
    ga, gb = torch.autograd.grad(residual_rms_norm(a, b, s["weight"], eps=EPS), (a, b), (dy, dh))
    assert torch.equal(g, ga + gb)


def test_rows_of_wider_tensors():
    s, dy, dh = inputs(40, 200, torch.bfloat16, torch.bfloat16, torch.bfloat16, True, "element")
    want = check(s, dy, dh)
    wide = {k: torch.nn.functional.pad(s[k], (3, 2))[:, 3:-2] for k in ("x", "residual", "gate")}
    got = check({**s, **wide}, *(torch.nn.functional.pad(t, (1, 4))[:, 1:-4] for t in (dy, dh)))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    assert all(torch.equal(want[2][k], got[2][k]) for k in want[2])
    turned = {k: s[k].t().contiguous().t() for k in ("x", "residual", "gate")}
    got = check({**s, **turned}, dy.t().contiguous().t(), dh)
    assert all(torch.equal(want[2][k], got[2][k]) for k in want[2])


def test_more_dimensions():
    x, r = torch.randn(2, 3, 4, 48, device=DEV).bfloat16(), torch.randn(2, 3, 4, 48, device=DEV)
    gate = torch.rand(2, 3, 4, 48, device=DEV).bfloat16()
    y, h = residual_rms_norm(x, r, gate=gate)
    y2, h2 = residual_rms_norm(x.view(24, 48), r.view(24, 48), gate=gate.view(24, 48))
    assert torch.equal(y.view(24, 48), y2) and torch.equal(h.view(24, 48), h2) and y.shape == x.shape


def test_gradient_against_differences():
    s, dy, dh = inputs(3, 21, torch.float32, torch.float32, torch.float32, True, "channel")
    s = {k: v.requires_grad_(True) for k, v in s.items()}
    names = list(s)
    grads = torch.autograd.grad(residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], residual_scale=0.5, eps=EPS),
                                [s[k] for k in names], (dy, dh))
    full = {k: v.detach().double().cpu() for k, v in s.items()}

    def value(x, residual, weight, post_weight, gate):
        n = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        h = 0.5 * residual + gate * n * post_weight
        y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * weight
        return ((y * dy.double().cpu()).sum() + (h * dh.double().cpu()).sum()).item()

    for k, g in zip(names, grads):
        flat = full[k].view(-1)
        for i in range(0, flat.numel(), 4):
            keep = flat[i].item()
            flat[i] = keep + 1e-5
            up = value(**full)
            flat[i] = keep - 1e-5
            down = value(**full)
            flat[i] = keep
            assert abs((up - down) / 2e-5 - g.view(-1)[i].item()) < 1e-4 * (1 + g.abs().max().item())


def test_more_than_2_32_bytes():
    """A block of rows again and again: the same bits in every copy, and the vectors' gradients as many times the block's."""
    copies, rows, cols = 140, 4000, 4096
    s, dy, dh = inputs(rows, cols, torch.bfloat16, torch.bfloat16, torch.float32, True, "channel")
    want = exact({k: v if v.dim() == 1 else v.double() for k, v in s.items()}, check(s, dy, dh)[1], dy, dh, 1.0)
    one = check(s, dy, dh)
    many = {k: v.repeat(copies, 1) if v.dim() == 2 else v for k, v in s.items()}
    assert many["x"].numel() * 2 > 1 << 32
    many = {k: v.requires_grad_(True) for k, v in many.items()}
    y, h = residual_rms_norm(many["x"], many["residual"], many["weight"], post_weight=many["post_weight"], gate=many["gate"], eps=EPS)
    grads = dict(zip(many, torch.autograd.grad((y, h), list(many.values()), (dy.repeat(copies, 1), dh.repeat(copies, 1)))))
    for c in range(copies):
        at = slice(c * rows, (c + 1) * rows)
        assert torch.equal(y[at], one[0]) and torch.equal(h[at], one[1])
        assert torch.equal(grads["x"][at], one[2]["x"]) and torch.equal(grads["residual"][at], one[2]["residual"])
    for k in ("weight", "post_weight", "gate"):
        # the bound of one block, whose sums are of copies times as many rows: a thread adds an eighth of the rows of a 256th of the chip, see exact()
        near(grads[k], copies * want[k][0], copies * (want[k][1] * copies), k)


def test_another_stream_and_twice_backward():
    s, dy, dh = inputs(257, 640, torch.bfloat16, torch.float32, torch.float32, True, "channel")
    s = {k: v.requires_grad_(True) for k, v in s.items()}

    def run():
        return residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], eps=EPS)

    want = run()
    grads = torch.autograd.grad(want, list(s.values()), (dy, dh), retain_graph=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run()
        back = torch.autograd.grad(got, list(s.values()), (dy, dh))
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*got, *back), (*want, *grads)))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, list(s.values()), (dy, dh)), grads))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(run(), want))


def test_nothing_to_do():
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    y, h = residual_rms_norm(x, x, w, post_weight=w, gate=w)
    assert y.shape == h.shape == (0, 16)
    got = torch.autograd.grad((y.sum(), h.sum()), (x, w))
    assert got[0].shape == (0, 16) and not got[1].any()


def test_rows_that_are_not_finite_stay_their_own():
    s, dy, dh = inputs(9, 128, torch.bfloat16, torch.bfloat16, torch.float32, True, "channel")
    clean = residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"])
    s["x"][4, 7] = float("nan")
    got = residual_rms_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"])
    keep = [i for i in range(9) if i != 4]
    assert all(torch.equal(a[keep], b[keep]) and torch.isnan(a[4]).all() for a, b in zip(got, clean))
    zero = torch.zeros(2, 128, device=DEV)
    y, h = residual_rms_norm(zero, zero, eps=1e-6)
    assert not y.any() and not h.any()


def test_module_and_graph():
    m = RMSNorm(256, device=DEV, post_norm=True, gate=True, gate_init=0.25, residual_scale=0.5)
    x, r = torch.randn(30, 256, device=DEV).bfloat16(), torch.randn(30, 256, device=DEV).bfloat16()
    dy, dh = torch.randn_like(x), torch.randn_like(r)
    leaves = [x.requires_grad_(True), r.requires_grad_(True), *m.parameters()]

    def step():
        y, h = m(x, r)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        with torch.no_grad():
            x.normal_()
            dy.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i
    with pytest.raises(ValueError, match="residual"):
        m(x)
    plain = RMSNorm(256, device=DEV)
    assert torch.equal(plain(x), rms_norm(x, plain.weight))


def test_refusals():
    x, w = torch.randn(4, 32, device=DEV).bfloat16(), torch.ones(32, device=DEV)
    for e, args, kw in ((TypeError, (x.double(), x, w), {}), (ValueError, (x, x[:3], w), {}), (TypeError, (x, x.half(), w), {}), (ValueError, (x, x, w[:31]), {}),
                        (TypeError, (x, x, w.half()), {}), (TypeError, (x, x, w), dict(post_weight=w.bfloat16())), (ValueError, (x, x, w), dict(gate=x[:2])),
                        (TypeError, (x, x, w), dict(gate=x.float())), (ValueError, (x, x, w), dict(eps=-1.0)), (ValueError, (x, x, w), dict(residual_scale=float("nan"))),
                        (ValueError, (x, x.cpu(), w), {}), (ValueError, (x, x, w.cpu()), {}), (TypeError, (x, x, w), dict(gate=w.bfloat16()))):
        with pytest.raises(e):
            residual_rms_norm(*args, **kw)
    with pytest.raises(ValueError, match="columns"):
        rms_norm(torch.zeros(1, 16385, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="columns"):
        rms_norm(torch.zeros(1, 8193, device=DEV))
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(rms_norm(leaf, w).float().sum(), leaf, create_graph=True)
