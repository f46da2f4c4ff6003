"""Layer normalisation against its formulas in 64 bits.

Tolerances.  With u = 2^-24 the fp32 passes bring, per element: the mean, a tree of sums over at most 2^15 elements, off by 32 u
mean|x| at most; xhat = (x - mean) rstd off by that times rstd and by 8 u |xhat| (difference, root, quotient, product; the
variance's own sums halved by the root).  The output adds u_out |y| of one rounding to its type (2^-24, 2^-11, 2^-8).
Gradients carry the error of xhat through sums of products, which are bounded by the sums of magnitudes."""
import pytest
import torch

from nanotron_amd.nn import LayerNorm, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def inputs(rows, cols, dtype, wdtype, shift=0.3, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) + shift * torch.randn(rows, 1, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(wdtype)
    b = (0.2 * torch.randn(cols, generator=g)).to(wdtype)
    dy = torch.randn(rows, cols, generator=g).to(dtype)
    return [t.to(DEV) for t in (x, w, b, dy)]


def exact(x, w, b, dy, eps):
    """(y, dx, dw, db), and bounds of what fp32 passes may be off by (before the rounding to the output's type)."""
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    n = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rstd
    ex = U32 * (32 * x.abs().mean(-1, keepdim=True) * rstd + 8 * xh.abs() + 32 * xh.abs())
    y = xh * w + b
    ey = ex * w.abs() + 2 * U32 * (xh * w).abs() + U32 * y.abs()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    a, h = g.abs(), xh.abs()
    # mean(g) and mean(g xh): sums of n terms in a tree, and xhat's own error; rstd is off by 40 u
    eg = 34 * U32 * a.mean(-1, keepdim=True)
    egx = 34 * U32 * (a * h).mean(-1, keepdim=True) + (a * ex).mean(-1, keepdim=True)
    inner = a + a.mean(-1, keepdim=True) + h * (a * h).mean(-1, keepdim=True)
    edx = rstd * (2 * U32 * a + eg + ex * (a * h).mean(-1, keepdim=True) + h * egx + 4 * U32 * inner) + 42 * U32 * rstd * inner
    rows = x.shape[0]
    # at most rows / 8 additions in a row in one thread, then 64 or fewer
    k = (min(rows, 4 + rows / 8) + 64) * U32
    dw, db = (dy * xh).sum(0), dy.sum(0)
    edw = (dy.abs() * ex).sum(0) + (k + 2 * U32) * (dy * xh).abs().sum(0)
    edb = k * dy.abs().sum(0)
    assert n > 0
    return (y, dx, dw, db), (ey, edx, edw, edb)


def near(got, want, bound, dtype, name):
    u = U[dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    off = (got.double() - want).abs()
    limit = bound + u * (want.abs() + bound) + tiny
    worst = (off / limit.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times what it may be off"


SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 63), (17, 512), (9, 513), (33, 1000), (64, 1024), (7, 1037), (130, 2048), (1021, 2049), (300, 4096),
          (5, 4097), (40, 8192), (3, 8191), (9, 16384)]


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_against_64_bits(rows, cols, dtype, wdtype):
    x, w, b, dy = inputs(rows, cols, dtype, wdtype)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = layer_norm(x, w, b)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    want, bound = exact(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    for o, a, e, n in zip(got, want, bound, ("y", "dx", "dweight", "dbias")):
        assert o.shape == a.shape and o.dtype == (wdtype if n[:2] in ("dw", "db") else dtype)
        near(o.detach(), a, e, o.dtype, n)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), y)


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 32768), (torch.bfloat16, 20001), (torch.float32, 16384), (torch.float32, 8200)])
def test_widest_rows(dtype, cols):
    x, w, b, dy = inputs(6, cols, dtype, torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = layer_norm(x, w, b)
    want, bound = exact(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    for o, a, e, n in zip((y, *torch.autograd.grad(y, (x, w, b), dy)), want, bound, ("y", "dx", "dweight", "dbias")):
        near(o.detach(), a, e, o.dtype, n)


def test_many_rows():
    x, w, b, dy = inputs(20011, 192, torch.bfloat16, torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    want, bound = exact(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    for o, a, e, n in zip((y, *grads), want, bound, ("y", "dx", "dweight", "dbias")):
        near(o.detach(), a, e, o.dtype, n)
    again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(weight, bias):
    x, w, b, dy = inputs(37, 640, torch.bfloat16, torch.float32)
    given = [w if weight else None, b if bias else None]
    leaves = [t.requires_grad_(True) for t in (x, *given) if t is not None]
    y = layer_norm(x, *given)
    grads = dict(zip(("x",) + ("w",) * weight + ("b",) * bias, torch.autograd.grad(y, leaves, dy)))
    want, bound = exact(x.detach(), w.detach() if weight else torch.ones_like(w), b.detach() if bias else torch.zeros_like(b), dy, 1e-5)
    near(y.detach(), want[0], bound[0], y.dtype, "y")
    for k, i in (("x", 1), ("w", 2), ("b", 3)):
        if k in grads:
            near(grads[k], want[i], bound[i], grads[k].dtype, k)


@pytest.mark.parametrize("leaf", [0, 1, 2])
def test_one_gradient_at_a_time(leaf):
    x, w, b, dy = inputs(50, 300, torch.float32, torch.float32)
    (x, w, b)[leaf].requires_grad_(True)
    y = layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b)[leaf], dy)[0]
    want, bound = exact(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    near(got, want[leaf + 1], bound[leaf + 1], got.dtype, "xwb"[leaf])


def test_gradient_against_differences():
    """The forward pass in 64 bits, differenced: an independent statement of the gradients (central differences are exact to h^2)."""
    x, w, b, dy = inputs(4, 33, torch.float32, torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)

    def value(x, w, b):
        mean = x.mean(-1, keepdim=True)
        return (((x - mean) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b) * dy.double()).sum()

    full = [t.detach().double() for t in (x, w, b)]
    h = 1e-5
    for i, g in enumerate(grads):
        flat = full[i].view(-1)
        for k in range(0, flat.numel(), 5):
            keep = flat[k].item()
            flat[k] = keep + h
            up = value(*full)
            flat[k] = keep - h
            down = value(*full)
            flat[k] = keep
            d = ((up - down) / (2 * h)).item()
            # differences of values ~ 100 in 64 bits: 1e-14 100 / h = 1e-7, the cubic term h^2 = 1e-10; the kernel's fp32 1e-5
            assert abs(g.view(-1)[k].item() - d) <= 2e-5 * (1 + abs(d))


def test_strides_shapes_and_other_streams():
    wide = torch.randn(60, 700, device=DEV, dtype=torch.bfloat16)
    w = torch.rand(500, device=DEV)
    inner = wide[:, 100:600]                                  # rows dense, 700 apart, on 2-byte boundaries
    odd = wide[:, 101:601]
    for x in (inner, odd, wide[::2, 3:503], wide.t()[100:600, :].t()):
        assert torch.equal(layer_norm(x, w), layer_norm(x.contiguous(), w))
        a, c = x.detach().requires_grad_(True), x.detach().contiguous().requires_grad_(True)
        dy = torch.randn(x.shape[0], 1400, device=DEV, dtype=torch.bfloat16)[:, 7:507]
        assert torch.equal(torch.autograd.grad(layer_norm(a, w), a, dy)[0], torch.autograd.grad(layer_norm(c, w), c, dy.contiguous())[0])
    x4 = wide.view(3, 4, 5, 700)
    assert torch.equal(layer_norm(x4).view(60, 700), layer_norm(wide))
    assert torch.equal(layer_norm(wide[0]), layer_norm(wide)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer_norm(inner, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, layer_norm(inner, w))


def test_large_means_and_specials():
    x = torch.randn(8, 2048, device=DEV) + 1000.0
    w, b = torch.ones(2048, device=DEV), torch.zeros(2048, device=DEV)
    want, bound = exact(x, w, b, x, 1e-5)
    near(layer_norm(x, w, b), want[0], bound[0], torch.float32, "y")
    assert (layer_norm(torch.full((3, 100), 7.0, device=DEV)) == 0).all()         # no variance: eps alone
    bad = torch.randn(4, 300, device=DEV, dtype=torch.bfloat16)
    bad[1, 17], bad[2, 299] = float("nan"), float("inf")
    y = layer_norm(bad)
    assert y[1].isnan().all() and y[2].isnan().all() and not y[0].isnan().any() and not y[3].isnan().any()


def test_no_rows():
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 64, device=DEV))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and (dw == 0).all()


def test_module_and_graph():
    m = LayerNorm(512, device=DEV)
    assert sum(p.numel() for p in m.parameters()) == 1024 and LayerNorm(8, elementwise_affine=False).weight is None and LayerNorm(8, bias=False).bias is None
    x = torch.randn(64, 512, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn_like(x)

    def step():
        y = m(x)
        return (y, *torch.autograd.grad(y, (x, m.weight, m.bias), dy))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), k


def test_refusals():
    x = torch.randn(4, 8, device=DEV)
    for bad, error in (((x.long(),), TypeError), ((x, torch.ones(7, device=DEV)), ValueError), ((x, torch.ones(8, device=DEV).half()), TypeError),
                       ((x, torch.ones(8)), ValueError), ((x, torch.ones(8, device=DEV), torch.ones(1, 8, device=DEV)), ValueError),
                       ((torch.randn(4, 0, device=DEV),), ValueError), ((torch.tensor(1.0, device=DEV),), ValueError), ((x, None, None, -1.0), ValueError)):
        with pytest.raises(error):
            layer_norm(*bad)
    with pytest.raises(RuntimeError, match="not supported"):
        layer_norm(torch.zeros(1, 40000, device=DEV, dtype=torch.bfloat16))


def test_differentiable_once():
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            layer_norm(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)))


def test_more_rows_than_a_launch_takes():
    """Rows of a few elements, more of them than threads of one launch can take (2^32, 64 a row)."""
    rows, cols = (1 << 26) + 1003, 3
    g = torch.Generator(device=DEV).manual_seed(2)
    x, dy = (torch.randn(rows, cols, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    w, b = (torch.randn(cols, generator=g, device=DEV) for _ in range(2))
    x.requires_grad_(True)
    y = layer_norm(x, w, b)
    y.backward(dy)
    # a launch ends at 2^21 workgroups of four rows each
    for first in (0, (1 << 23) - 500, (1 << 25) - 500, rows - 1000):
        part = slice(first, first + 1000)
        want, bound = exact(x.detach()[part], w, b, dy[part], 1e-5)
        near(y.detach()[part], want[0], bound[0], y.dtype, "y")
        near(x.grad[part], want[1], bound[1], x.dtype, "dx")


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes of x: the last rows are those of the formulas."""
    rows, cols = 270001, 8192
    g = torch.Generator(device=DEV).manual_seed(3)
    x, dy = (torch.randn(rows, cols, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    w, b = (torch.randn(cols, generator=g, device=DEV) for _ in range(2))
    x.requires_grad_(True)
    y = layer_norm(x, w, b)
    y.backward(dy)
    assert x.numel() * 2 > 1 << 32
    for part in (slice(0, 100), slice(rows // 2 - 50, rows // 2 + 50), slice(rows - 100, rows)):
        want, bound = exact(x.detach()[part], w, b, dy[part], 1e-5)
        near(y.detach()[part], want[0], bound[0], y.dtype, "y")
        near(x.grad[part], want[1], bound[1], x.dtype, "dx")
    del x, y, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [1000, 7168, 100, 33, 16384])
def test_constant_rows(cols, dtype):
    """Rows of one value have no deviation at all, whatever the value and their length: exactly the bias comes out.  (The sum may
    round, and the mean with it, to a neighbour of the value at most; the sum of the differences from that is small whole
    multiples of an ulp, exact, and so is its quotient.)"""
    values = torch.tensor([1000.0, 100.0, 1000.1, 3.3, -17.77, 0.1, 1e-3, 60000.0, 1 / 3, 0.0], device=DEV).to(dtype)
    x = values[:, None].expand(-1, cols).contiguous()
    b = torch.randn(cols, device=DEV)
    assert (layer_norm(x) == 0).all()
    assert torch.equal(layer_norm(x, torch.full((cols,), 3.0, device=DEV), b), b.to(dtype).expand(len(values), -1))
    # backward: xhat is 0, dx = rstd (g - mean g)
    x.requires_grad_(True)
    w = torch.ones(cols, device=DEV, requires_grad=True)
    dy = torch.randn(len(values), cols, device=DEV).to(dtype)
    dx, dw = torch.autograd.grad(layer_norm(x, w), (x, w), dy)
    assert (dw == 0).all()
    d = dy.double()
    want = (d - d.mean(-1, keepdim=True)) / 1e-5 ** 0.5
    # mean(g): a tree of sums, 34 u mean|g|; a difference, a product, rstd (4 u)
    near(dx, want, U32 / 1e-5 ** 0.5 * (34 * d.abs().mean(-1, keepdim=True) + 6 * (d.abs() + d.abs().mean(-1, keepdim=True))), dtype, "dx")


def test_weight_gradient_of_rows_that_cancel():
    """Two rows of dy of 2^27 that cancel, among 1019 of ones.  In 32 bits a value passes the additions in its thread and its
    workgroup only (two rows a thread and two threads of a column here, three additions with the one onto zero, which is exact);
    everything behind them is summed in 64.  Of four additions at 2^27 each is off by half of 16 at most."""
    rows, cols = 1021, 1037
    x = torch.randn(rows, cols, device=DEV)
    dy = torch.ones(rows, cols, device=DEV)
    dy[0], dy[-1] = 2.0 ** 27, -2.0 ** 27
    w, b = torch.ones(cols, device=DEV, requires_grad=True), torch.zeros(cols, device=DEV, requires_grad=True)
    y = layer_norm(x, w, b)
    db, = torch.autograd.grad(y, b, dy, retain_graph=True)
    assert ((db - (rows - 2)).abs() <= 4 * 8).all()
    # the same of xhat: rows 0 and last alike, and bounded entries (xhat of two values, +-1 but for eps)
    x = torch.ones(rows, cols - 1, device=DEV)
    x[:, ::2] = -1.0
    y = layer_norm(x, w[:-1])
    dw, = torch.autograd.grad(y, w, dy[:, :-1])
    xh = torch.where(torch.arange(cols - 1, device=DEV) % 2 == 0, -1.0, 1.0).double() / (1 + 1e-5) ** 0.5
    # (4 additions, and the product's own rounding of the two large ones, which are alike and cancel)
    assert ((dw[:-1] - (rows - 2) * xh).abs() <= 4 * 8 + 1e-3).all()


@pytest.mark.parametrize("rows,cols", [(11, 200), (7, 1000), (9, 1500), (6, 4000), (5, 8192), (4, 16384)])
def test_rows_far_from_zero(rows, cols):
    """Every other row 1000 deviations from zero, beside ordinary ones.  There the mean's own error is taken out: a difference is exact
    or off by u, the rest of the mean by 32 u of a deviation, rstd by 36 u."""
    x, w, b, dy = inputs(rows, cols, torch.float32, torch.float32, seed=cols)
    x[::2] += 1000.0
    want, bound = exact(x, w, b, dy, 1e-5)
    y = layer_norm(x, w, b)
    near(y, want[0], bound[0], torch.float32, "y")
    xd = x.double()
    xh = (xd - xd.mean(-1, keepdim=True)) * (xd.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    far = U32 * (32 + 40 * xh.abs()) * w.double().abs() + 2 * U32 * (xh * w.double()).abs() + U32 * want[0].abs()
    near(y[::2], want[0][::2], far[::2], torch.float32, "y of the rows far from zero")
