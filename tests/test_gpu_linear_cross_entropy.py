"""The projection's softmax cross entropy against its formulas in 64 bits.

Tolerances, u = 2^-24.  A logit is a sum of `hidden` exact products: off by (hidden / 32 + 40) u sum|x w| at most (the matrix
core adds 32 products at a time); call the largest of a row e.  A loss is off by 2 e and 8 u of its terms.  An entry of dl, the softmax
minus the label's one, carries 2 e + 40 u from the softmax, 2^-11 of its kept exponential and one rounding to the
inputs' type (2^-8 bf16, 2^-11 fp16); exponentials 2^-29 below their piece's maximum lose bits, 2^-40 in all.  dx and
dweight are sums of such entries times inputs, bounded with the magnitudes' own products, and are rounded to their type."""
import pytest
import torch

from nanotron_amd import _native as nt
from nanotron_amd import _ops
from nanotron_amd.nn import LinearCrossEntropy, linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24


def draw(tokens, hidden, vocab, dtype, ignored=0.0, seed=0, lean=4.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(vocab, hidden, generator=g, device=DEV) * (1.3 / hidden ** 0.5)).to(dtype)
    labels = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    x = (torch.randn(tokens, hidden, generator=g, device=DEV) + lean * torch.rand(tokens, 1, generator=g, device=DEV) * w[labels].float()).to(dtype)
    if ignored:
        labels = torch.where(torch.rand(tokens, generator=g, device=DEV) < ignored, -100, labels)
    return x, w, labels


def exact(x, w, labels, mean=True):
    """losses, loss, dx, dw and their bounds before the outputs' own rounding."""
    ut = UT[x.dtype]
    x, w = x.double(), w.double()
    logits = x @ w.t()
    e = ((x.shape[1] / 32 + 40) * U32 * (x.abs() @ w.abs().t()).amax(-1))
    keep = labels != -100
    at = torch.where(keep, labels, 0)
    lse = torch.logsumexp(logits, -1)
    losses = torch.where(keep, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    el = torch.where(keep, 2 * e + 8 * U32 * (lse.abs() + losses.abs() + 20), 0.0)
    f = 1.0 / max(1, int(keep.sum())) if mean else 1.0
    p = torch.softmax(logits, -1)
    dl = p.clone()
    dl[torch.arange(len(at)), at] -= 1
    dl, p = dl * keep[:, None], p * keep[:, None]
    share = (2 * e + 40 * U32)[:, None]
    edl = share * p + (2.0 ** -11 + ut) * dl.abs() + 2.0 ** -40
    n = x.shape[0]
    dx, dw = f * (dl @ w), f * (dl.t() @ x)
    a = dl.abs() + edl
    edx = f * (edl @ w.abs() + (w.shape[0] / 32 + 300) * U32 * (a @ w.abs())) + 2 * U32 * dx.abs()
    edw = f * (edl.t() @ x.abs() + (n / 32 + 300) * U32 * (a.t() @ x.abs())) + 2 * U32 * dw.abs()
    total = losses.sum() * f
    return (losses, total, dx, dw), (el, f * el.sum() + (n / 1024 + 30) * U32 * f * losses.abs().sum(), edx, edw)


def near(got, want, bound, name):
    u = UT.get(got.dtype, U32)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -130
    worst = ((got.double() - want).abs() / (bound + u * (want.abs() + bound) + tiny)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times what it may be off"


def check(x, w, labels, reduction="mean"):
    want, bound = exact(x, w, labels, reduction == "mean")
    with torch.no_grad():
        losses = linear_cross_entropy(x, w, labels, reduction="none")
        alone = linear_cross_entropy(x, w, labels, reduction=reduction)
    assert losses.shape == labels.shape and losses.dtype == torch.float32
    near(losses, want[0], bound[0], "losses")
    near(alone, want[1], bound[1], "loss")
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(a, b, labels, reduction=reduction)
    loss.backward()
    near(loss.detach(), want[1], bound[1], "loss")
    assert a.grad.dtype == x.dtype and b.grad.dtype == w.dtype
    near(a.grad, want[2], bound[2], "dx")
    near(b.grad, want[3], bound[3], "dweight")


SIZES = [(1, 8, 1), (1, 64, 2), (2, 8, 9), (3, 515, 601), (16, 256, 1000), (31, 130, 257), (33, 64, 4099), (64, 1024, 128), (65, 72, 3001), (128, 512, 8000),
         (129, 520, 777), (200, 96, 65), (333, 515, 6001), (256, 256, 256), (257, 264, 511), (600, 1024, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hidden,vocab", SIZES)
def test_against_64_bits(tokens, hidden, vocab, dtype):
    check(*draw(tokens, hidden, vocab, dtype, 0.2 if tokens > 8 else 0.0, tokens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sum_and_large_vocabulary(dtype):
    check(*draw(70, 128, 50001, dtype, 0.3, 5), reduction="sum")


@pytest.mark.parametrize("tokens,hidden,vocab", [(700, 136, 40000), (520, 512, 30001), (1100, 64, 25000), (300, 1000, 52001)])
def test_large_tiles(tokens, hidden, vocab):
    """Sizes whose products are made of 256-row tiles, several to a workgroup: one K-tile and many, and K-tiles that end inside."""
    check(*draw(tokens, hidden, vocab, torch.bfloat16, 0.2, 8))
    check(*draw(tokens, hidden, vocab, torch.float16, 0.0, 9))


def test_long_batch():
    check(*draw(2500, 256, 1501, torch.bfloat16, 0.1, 6))


def test_sharp_and_flat_rows():
    """Certain predictions (the label's probability 1 - 1e-6 and less), equal logits, a row far from its label."""
    x, w, labels = draw(64, 256, 3000, torch.bfloat16, 0.0, 7, lean=0.0)
    x[:16] = (x[:16].float() * 0.1 + 20 * w[labels[:16]].float()).bfloat16()
    x[16:32] = 0
    x[32:48] = (-20 * w[labels[32:48]].float()).bfloat16()
    check(x, w, labels)
    # all tokens right for certain: gradients next to nothing, losses exact to fp32
    check(x[:16], w, labels[:16])


def test_all_rows_ignored():
    x, w, _ = draw(40, 64, 500, torch.bfloat16)
    labels = torch.full((40,), -100, device=DEV)
    x[3, 5] = float("nan")      # in an ignored token: nobody sees it
    for reduction in ("mean", "sum"):
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(a, b, labels, reduction=reduction)
        loss.backward()
        assert loss.item() == 0 and (a.grad == 0).all() and (b.grad == 0).all()
    with torch.no_grad():
        assert (linear_cross_entropy(x, w, labels, reduction="none") == 0).all()


def test_another_ignore_index_and_shapes():
    x, w, labels = draw(60, 64, 300, torch.bfloat16, 0.0, 9)
    labels[::3] = 0
    other = torch.where(labels == 0, -100, labels)
    with torch.no_grad():
        a = linear_cross_entropy(x.view(3, 4, 5, 64), w, labels.view(3, 4, 5), ignore_index=0, reduction="none")
        b = linear_cross_entropy(x, w, other, reduction="none")
        assert a.shape == (3, 4, 5) and torch.equal(a.view(-1), b)
        assert torch.equal(linear_cross_entropy(x, w, labels, ignore_index=0), linear_cross_entropy(x, w, other))


@pytest.mark.parametrize("bad", [300, 301, 511, 1 << 40, -1, -(1 << 40)])
def test_label_outside_the_vocabulary(bad):
    x, w, labels = draw(50, 64, 300, torch.bfloat16, 0.0, 10)
    good = linear_cross_entropy(x, w, labels, reduction="none")
    labels[7] = bad
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(a, b, labels)
    loss.backward()
    assert loss.isnan() and a.grad[7].isnan().all() and not a.grad[8].isnan().any()
    with torch.no_grad():
        got = linear_cross_entropy(x, w, labels, reduction="none")
    assert got[7].isnan() and torch.equal(got[8:], good[8:])


def test_specials():
    x, w, labels = draw(40, 64, 700, torch.bfloat16, 0.0, 11)
    x[4, 3], x[9, 1] = float("nan"), float("inf")
    got = linear_cross_entropy(x, w, labels, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[4] = bad[9] = True
    assert torch.equal(got.isnan(), bad)
    # rows of -inf and +inf logits for some columns: a column of -inf has no weight
    x, w, labels = draw(8, 64, 700, torch.float16, 0.0, 12)
    x.abs_()
    w[50:400] = -60000.0
    w[400] = 0
    x = (x + 20).half()
    logits = (x.float() @ w.float().t())
    labels[:] = 500
    ref = torch.logsumexp(logits.double(), -1) - logits[:, 500].double()
    got = linear_cross_entropy(x, w, labels, reduction="none")
    assert ((got - ref).abs() <= 1e-4 * (1 + logits.abs()[:, 500:].amax(-1))).all()


def test_gradient_against_differences():
    """The loss in 64 bits, differenced along random directions of x and weight."""
    x, w, labels = draw(24, 72, 130, torch.float16, 0.2, 13)
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    linear_cross_entropy(a, b, labels).backward()
    want, bound = exact(x, w, labels)
    g = torch.Generator(device=DEV).manual_seed(3)

    def loss(x, w):
        return torch.nn.functional.cross_entropy(x @ w.t(), labels)

    h = 1e-4
    for _ in range(8):
        dx, dw = (torch.randn(t.shape, generator=g, device=DEV, dtype=torch.float64) for t in (x, w))
        d = (loss(x.double() + h * dx, w.double() + h * dw) - loss(x.double() - h * dx, w.double() - h * dw)) / (2 * h)
        got = (a.grad.double() * dx).sum() + (b.grad.double() * dw).sum()
        limit = ((bound[2] + 2.0 ** -11 * want[2].abs() + 2.0 ** -25) * dx.abs()).sum() + ((bound[3] + 2.0 ** -11 * want[3].abs() + 2.0 ** -25) * dw.abs()).sum()
        assert (got - d).abs() <= limit + 1e-5 * d.abs() + 1e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_upstream_gradient(dtype):
    x, w, labels = draw(100, 128, 900, dtype, 0.1, 14)
    want, bound = exact(x, w, labels)
    for factor in (1.0, 0.25, 3.0, 1024.0):
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        (linear_cross_entropy(a, b, labels) * factor).backward()
        # (a bf16 gradient is rounded, multiplied and rounded again)
        for got, i, name in ((a.grad, 2, "dx"), (b.grad, 3, "dweight")):
            near(got, want[i] * factor, (bound[i] + UT[dtype] * want[i].abs()) * factor, name)


def test_one_gradient_at_a_time_and_accumulation():
    x, w, labels = draw(90, 128, 700, torch.bfloat16, 0.1, 15)
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    linear_cross_entropy(a, b, labels).backward()
    c, d = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    linear_cross_entropy(c, w, labels).backward()
    linear_cross_entropy(x, d, labels).backward()
    assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)
    first = d.grad.clone()
    linear_cross_entropy(x, d, labels).backward()
    assert torch.equal(d.grad, first + first)
    loss = linear_cross_entropy(a, b, labels)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        loss.backward()


def test_strides_and_streams():
    x, w, labels = draw(100, 256, 800, torch.bfloat16, 0.1, 16)
    wide_x, wide_w = torch.randn(100, 400, device=DEV).bfloat16(), torch.randn(800, 300, device=DEV).bfloat16()
    with torch.no_grad():
        want = linear_cross_entropy(x, w, labels, reduction="none")
    for at in (0, 8, 3):     # rows on 16-byte boundaries, and not
        wide_x[:, at:at + 256], wide_w[:, at:at + 256] = x, w
        a, b = wide_x[:, at:at + 256].detach().requires_grad_(True), wide_w[:, at:at + 256].detach().requires_grad_(True)
        loss = linear_cross_entropy(a, b, labels)
        loss.backward()
        c, d = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        linear_cross_entropy(c, d, labels).backward()
        assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        got = linear_cross_entropy(x.t().contiguous().t(), w, labels, reduction="none")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_graph_replays():
    x, w, labels = draw(150, 128, 3000, torch.bfloat16, 0.1, 17)
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)

    def step():
        loss = linear_cross_entropy(a, b, labels)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b)))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x2, w2, l2 = draw(150, 128, 3000, torch.bfloat16, 0.2, 30 + k)
            a.copy_(x2), b.copy_(w2), labels.copy_(l2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step())), k


@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, nt.BF16), (torch.float16, nt.F16)])
def test_tokens_in_pieces(dtype, code):
    """More tokens than go at a time: the weight's gradient is collected in fp32.  The vocabulary of 2^22 makes pieces of
    256 tokens, too large a test; a narrow hidden size keeps this one small."""
    vocab = 1 << 21
    piece = _ops.lib.ntops_linear_cross_entropy_piece(vocab)
    assert piece == 512
    tokens = piece + 40
    x, w, labels = draw(tokens, 16, vocab, dtype, 0.1, 18)
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(a, b, labels)
    loss.backward()
    # 64 bits in runs of tokens
    keep = labels != -100
    f = 1.0 / int(keep.sum())
    total, dw, bw = 0.0, torch.zeros(vocab, 16, device=DEV, dtype=torch.float64), torch.zeros(vocab, 16, device=DEV, dtype=torch.float64)
    for r in range(0, tokens, 138):
        part = slice(r, min(tokens, r + 138))
        want, bound = exact(x[part], w, labels[part], mean=False)
        near(a.grad[part], want[2] * f, bound[2] * f, "dx")
        total += want[0].sum().item() * f
        dw += want[3] * f
        bw += bound[3] * f
    near(b.grad, dw, bw, "dweight")
    assert abs(loss.item() - total) <= 1e-5 * total


def test_module_and_empty_batch():
    m = LinearCrossEntropy(64, 500, device=DEV)
    x = torch.randn(2, 10, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    labels = torch.randint(0, 500, (2, 10), device=DEV)
    m(x, labels).backward()
    assert m.weight.grad.shape == (500, 64) and x.grad.shape == x.shape
    m.weight.grad = None
    e = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    loss = m(e, torch.empty(0, device=DEV, dtype=torch.int64))
    loss.backward()
    assert loss.item() == 0 and (m.weight.grad == 0).all()
    with torch.no_grad():
        assert linear_cross_entropy(e, m.weight, torch.empty(0, device=DEV, dtype=torch.int64), reduction="none").shape == (0,)


def test_refusals():
    x, w, labels = draw(10, 64, 100, torch.bfloat16)
    for args, kw, error in (((x.float(), w.float(), labels), {}, TypeError), ((x, w.half(), labels), {}, TypeError), ((x, w, labels.int()), {}, TypeError),
                            ((x, w[:, :63], labels), {}, ValueError), ((x, w, labels[:9]), {}, ValueError), ((x, w.cpu(), labels), {}, ValueError),
                            ((x, w, labels), dict(reduction="max"), ValueError), ((x.requires_grad_(True), w, labels), dict(reduction="none"), ValueError)):
        with pytest.raises(error):
            linear_cross_entropy(*args, **kw)


def test_differentiable_once():
    x, w, labels = draw(10, 64, 100, torch.bfloat16)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(linear_cross_entropy(x, w, labels), x, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            linear_cross_entropy(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)), w, labels)


def test_losses_in_pieces():
    """Losses alone, of more tokens than are taken at a time."""
    vocab = 1 << 21
    tokens = (1 << 31) // (8 * (vocab // 128)) + 300
    x, w, labels = draw(tokens, 8, vocab, torch.bfloat16, 0.1, 19)
    got = linear_cross_entropy(x, w, labels, reduction="none")
    for r in (0, 5000, tokens - 301, tokens - 40):
        part = slice(r, r + 40)
        want, bound = exact(x[part], w, labels[part])
        near(got[part], want[0], bound[0], "losses")


def test_many_tokens_of_few_labels():
    """More tokens than a launch with a token to a workgroup takes."""
    tokens = (1 << 24) + 300
    x, w, labels = draw(tokens, 8, 5, torch.bfloat16, 0.1, 20)
    x.requires_grad_(True)
    linear_cross_entropy(x, w, labels, reduction="sum").backward()
    with torch.no_grad():
        losses = linear_cross_entropy(x, w, labels, reduction="none")
    for first in (0, (1 << 23) - 500, (1 << 24) - 500, tokens - 1000):
        part = slice(first, first + 1000)
        want, bound = exact(x.detach()[part], w, labels[part], mean=False)
        near(losses[part], want[0], bound[0], "losses")
        near(x.grad[part], want[2], bound[2], "dx")


def test_offsets_beyond_32_bits():
    """A weight of more than 2^32 bytes, in 64 bits by runs of its rows."""
    tokens, hidden, vocab, run = 40, 4096, (1 << 19) + 4099, 1 << 15
    x, w, labels = draw(tokens, hidden, vocab, torch.bfloat16, 0.1, 21)
    labels[:4] = torch.tensor([0, vocab - 1, vocab - 2, 1 << 19], device=DEV)
    assert w.numel() * 2 > 1 << 32
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(a, b, labels, reduction="sum")
    loss.backward()
    xd, ut = x.double(), UT[x.dtype]
    runs = [slice(r, min(vocab, r + run)) for r in range(0, vocab, run)]
    logits = torch.cat([xd @ w[r].double().t() for r in runs], 1)
    e = (hidden / 32 + 40) * U32 * torch.stack([(xd.abs() @ w[r].double().abs().t()).amax(-1) for r in runs]).amax(0)
    keep = labels != -100
    at = torch.where(keep, labels, 0)
    lse = torch.logsumexp(logits, -1)
    losses = torch.where(keep, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    near(loss.detach(), losses.sum(), (2 * e + 8 * U32 * (lse.abs() + losses.abs() + 20)).sum(), "loss")
    p = torch.softmax(logits, -1)
    dl = p.clone()
    dl[torch.arange(tokens), at] -= 1
    dl, p = dl * keep[:, None], p * keep[:, None]
    edl = (2 * e + 40 * U32)[:, None] * p + (2.0 ** -11 + ut) * dl.abs() + 2.0 ** -40
    dx, edx = torch.zeros_like(xd), torch.zeros_like(xd)
    for r in runs:
        wr = w[r].double()
        dx += dl[:, r] @ wr
        edx += edl[:, r] @ wr.abs() + (vocab / 32 + 300) * U32 * ((dl[:, r].abs() + edl[:, r]) @ wr.abs())
    near(a.grad, dx, edx + 2 * U32 * dx.abs(), "dx")
    for r in (slice(0, 1000), slice((1 << 19) - 500, (1 << 19) + 500), slice(vocab - 1000, vocab)):
        dw = dl[:, r].t() @ xd
        near(b.grad[r], dw, edl[:, r].t() @ xd.abs() + (tokens / 32 + 300) * U32 * ((dl[:, r].abs() + edl[:, r]).t() @ xd.abs()) + 2 * U32 * dw.abs(), "dweight")
    del a, b, x, w
    torch.cuda.empty_cache()


def test_no_tokens_beside_a_weight_that_is_not_finite():
    x = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = torch.full((500, 64), float("inf"), device=DEV, dtype=torch.bfloat16, requires_grad=True)
    loss = linear_cross_entropy(x, w, torch.empty(0, device=DEV, dtype=torch.int64))
    loss.backward()
    assert loss.dtype == torch.float32 and loss.item() == 0.0
    assert x.grad.shape == x.shape and not w.grad.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_far_apart(dtype):
    """The last token of every sequence of a long batch, and a weight whose rows lie as far apart: more than 2^22 elements."""
    hidden, length, vocab = 4096, 1031, 33
    h = torch.zeros(5, length, hidden, device=DEV, dtype=dtype)
    x, w, labels = draw(5, hidden, vocab, dtype, 0.0, 24)
    labels[3] = -100
    h[:, -1] = x
    wide = torch.zeros(vocab, (1 << 22) + 8, device=DEV, dtype=dtype)
    wide[:, 8:8 + hidden] = w
    assert h[:, -1].stride(0) > 1 << 22 and wide.stride(0) > 1 << 22
    for rows, weight in ((h[:, -1], w), (x, wide[:, 8:8 + hidden]), (h[:, -1], wide[:, 8:8 + hidden])):
        check(rows, weight, labels)
        with torch.no_grad():
            assert torch.equal(linear_cross_entropy(rows, weight, labels, reduction="none"), linear_cross_entropy(x, w, labels, reduction="none"))
    del h, wide
    torch.cuda.empty_cache()


@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_dx_in_pieces_of_its_own(reduction):
    """So many tokens of so few labels that all logits are held at once and the sums of dx are not: its rows on both sides
    of where a piece ends (2^31 bytes of sums, 65280 rows here), ignored ones among them, and the weight's whole gradient."""
    tokens, hidden, vocab = 70001, 8200, 301
    x, w, labels = draw(tokens, hidden, vocab, torch.bfloat16, 0.05, 23)
    a, b = x.requires_grad_(True), w.requires_grad_(True)
    linear_cross_entropy(a, b, labels, reduction=reduction).backward()
    x, w = x.detach(), w.detach()
    count = int((labels != -100).sum())
    f = 1.0 / count if reduction == "mean" else 1.0
    assert 65280 < count < 65280 + 2000
    dw, bw = torch.zeros(vocab, hidden, device=DEV, dtype=torch.float64), torch.zeros(vocab, hidden, device=DEV, dtype=torch.float64)
    for r in range(0, tokens, 10000):
        part = slice(r, min(tokens, r + 10000))
        want, bound = exact(x[part], w, labels[part], mean=False)
        near(a.grad[part], want[2] * f, bound[2] * f, f"dx of {r}")
        dw += want[3] * f
        bw += bound[3] * f
    near(b.grad, dw, bw, "dweight")
    del a, b, x, w, dw, bw
    torch.cuda.empty_cache()
