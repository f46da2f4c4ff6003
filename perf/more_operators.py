"""Measured cases of the operators between a decoder layer's linears: attention, rotary positions, and the norms around a block
with its gate and residual.

Every case is a dict of plain values.  `kind` says which operator it calls:

  attention   softmax(scale q k^T) v with grouped heads over sequences of different lengths laid end to end (`sequences` of them in
              `tokens` rows), forward and backward; or, with `context`, the last `tokens` rows of each of `batch` sequences against a
              cache of `context` keys, forward alone.  Causal rows see the keys up to their own, counted from the sequence's end
  rotary      rotation of the first `part` elements of every query and key head by angles position * frequency, pairs side by side
              (`interleaved`) or half of the part apart; frequencies plain or scaled for longer contexts
  norms       h = residual_scale residual + gate * norm(x) post_weight, y = norm(h) weight, with norm(x) = x / root(mean(x^2) + eps);
              the norm behind the block (`post`) and the gate (one value a channel, or one an element) may be absent

With `own` false, `run` computes them in 32 bits (angles in 64) from elementary torch operations.  Sizes: heads, hidden size and
tokens of this repository's benchmark layer (32 query heads and 8 key heads of 128 in 4096), sizes of its tests, and generic ones.
"""
import math

import torch

own = False

DEVICE = torch.device("cuda", 0)
TORCH = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6
SCORES = 1 << 28     # elements of a matrix of scores that the plain form holds at once


def listed():
    return [
        # one new token of one request over its cache: launch and host time
        dict(name="attention 1 token over 4096", kind="attention", batch=1, tokens=1, context=4096, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # one new token of many requests: the cache is read once
        dict(name="attention 32 tokens over 8192", kind="attention", batch=32, tokens=1, context=8192, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # a piece of a long prompt behind what is in the cache already
        dict(name="attention prompt 512 over 8192", kind="attention", batch=1, tokens=512, context=8192, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # a small model's step on documents packed end to end, lengths that are multiples of nothing
        dict(name="attention step 3001 packed fp16", kind="attention", tokens=3001, sequences=13, heads=12, kv_heads=4, dim=64, dtype="fp16", causal=True),
        # an encoder's batch: every token sees its whole sequence, heads of a size between the tiles'
        dict(name="attention step 4999 both ways", kind="attention", tokens=4999, sequences=9, heads=16, kv_heads=16, dim=80, dtype="bf16", causal=False),
        # the benchmark layer
        dict(name="attention step 4096", kind="attention", tokens=4096, sequences=1, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # a long context through the same layer
        dict(name="attention step 16384", kind="attention", tokens=16384, sequences=1, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True),
        # queries and key of one new token
        dict(name="rotary 1 token", kind="rotary", tokens=1, heads=32, kv_heads=8, dim=128, part=128, dtype="bf16", interleaved=False, scaling="none", far=4096, train=False),
        # a long batch through part of each head, positions beyond those a model was made for
        dict(name="rotary step 16381 scaled", kind="rotary", tokens=16381, heads=32, kv_heads=8, dim=128, part=96, dtype="bf16", interleaved=True, scaling="yarn", far=131072, train=True),
        # between two blocks for one token
        dict(name="norms 1 token", kind="norms", rows=1, cols=4096, dtype="bf16", rdtype="bf16", wdtype="bf16", post=False, gate="none", scale=1.0, train=False),
        # sizes that are multiples of nothing, every part there, a gate for each element
        dict(name="norms step 1021x1037 fp16", kind="norms", rows=1021, cols=1037, dtype="fp16", rdtype="fp16", wdtype="fp16", post=True, gate="element", scale=0.5, train=True),
        # a long batch, norms before and after each block, a residual stream in 32 bits
        dict(name="norms step 16384x4096 both", kind="norms", rows=16384, cols=4096, dtype="bf16", rdtype="fp32", wdtype="fp32", post=True, gate="channel", scale=1.0, train=True),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, grid=1):
    """A size between lo and hi, spread over its logarithm, on a grid where it is large enough for it."""
    v = int(_log(rng, lo, hi + 0.99))
    return max(lo, min(hi, v // grid * grid if v >= grid else v))


def _scaling(rng):
    return rng.choice(["none", "none", "linear", "yarn"])


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "rotary", "norms"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    dim = rng.choice([64, 80, 96, 128, 128])
    grid = rng.choice([128, 1])
    if kind == "rotary":
        return dict(kind=kind, tokens=_size(rng, 1, 16384, grid), heads=heads, kv_heads=kv_heads, dim=dim, part=rng.choice([dim, dim // 2]), dtype=dtype,
                    interleaved=rng.random() < 0.5, scaling=_scaling(rng), far=_size(rng, 2048, 131072), train=rng.random() < 0.6)
    if kind == "norms":
        rdtype = rng.choice([dtype, dtype, "fp32"])
        return dict(kind=kind, rows=_size(rng, 1, 16384, grid), cols=_size(rng, 64, 4096, rng.choice([128, 16, 1])), dtype=dtype, rdtype=rdtype,
                    wdtype=rng.choice([dtype, "fp32"]), post=rng.random() < 0.5, gate=rng.choice(["none", "channel", "element"]),
                    scale=rng.choice([1.0, 1.0, 0.5]), train=rng.random() < 0.7)
    what = rng.choice(["step", "step", "tokens", "prompt"])
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    if what == "step":
        tokens = _size(rng, 64, 8192, grid)
        return dict(c, tokens=tokens, sequences=_size(rng, 1, max(1, min(40, tokens // 8))), causal=rng.random() < 0.8)
    if what == "tokens":
        context = _size(rng, 1, 32768)
        return dict(c, batch=_size(rng, 1, max(1, min(64, (1 << 28) // (context * kv_heads * dim)))), tokens=1, context=context, causal=True)
    context = _size(rng, 512, 16384, grid)
    return dict(c, batch=rng.choice([1, 1, 2, 3]), tokens=min(context, _size(rng, 2, 1024, grid)), context=context, causal=rng.random() < 0.9)


def _lengths(case):
    """Lengths of the packed sequences: uneven, of any size from nothing up."""
    n, total = case["sequences"], case["tokens"]
    cuts = sorted(int(total * (i * 0.6180339887498949 % 1.0) ** 1.5) for i in range(1, n))
    ends = cuts + [total]
    return [b - a for a, b in zip([0] + cuts, ends)]


def _pairs(case):
    """Pairs of a query and a key that it sees."""
    if "context" in case:
        n, m = case["tokens"], case["context"]
        return case["batch"] * (n * m - (n * (n - 1) // 2 if case["causal"] else 0))
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, shape, std, dtype):
    return (torch.randn(shape, generator=g, device=DEVICE) * std).to(dtype)


def _frequencies(part, scaling, far):
    """(frequencies of the pairs, factor of sine and cosine), a model made for contexts of 8192 stretched to `far`."""
    base, made, factor = 500000.0, 8192, max(1.0, far / 8192)
    f = [base ** (-2.0 * i / part) for i in range(part // 2)]
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if scaling == "yarn":
        # pairs that turn less than once over the context are stretched, those that turn more than 32 times stay, a ramp between
        def pair(turns):
            return part * math.log(made / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(0, math.floor(pair(32.0))), min(part - 1, math.ceil(pair(1.0)))
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(part // 2)]
        return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    dt = TORCH[case["dtype"]]
    if case["kind"] == "norms":
        rows, cols, rd, wd = case["rows"], case["cols"], TORCH[case["rdtype"]], TORCH[case["wdtype"]]
        level = 0.2 + 2 * torch.rand((rows, 1), generator=g, device=DEVICE)
        residual = torch.randn((rows, cols), generator=g, device=DEVICE) * (1 + 8 * (torch.rand(cols, generator=g, device=DEVICE) < 0.01))
        s.update(x=(torch.randn((rows, cols), generator=g, device=DEVICE) * level).to(dt), residual=residual.to(rd), post_weight=None, channel=None,
                 weight=(1 + _normal(g, (cols,), 0.1, torch.float32)).to(wd))
        if case["post"]:
            s["post_weight"] = (0.5 + _normal(g, (cols,), 0.1, torch.float32)).to(wd)
        if case["gate"] == "channel":
            s["channel"] = (0.3 + _normal(g, (cols,), 0.1, torch.float32)).to(wd)
        if case["gate"] == "element":
            s["channel"] = torch.sigmoid(torch.randn((rows, cols), generator=g, device=DEVICE)).to(dt)
        s["leaves"] = [k for k in ("x", "residual", "weight", "post_weight", "channel") if s[k] is not None]
        if case["train"]:
            s.update(dy=_normal(g, (rows, cols), 1e-1, dt), dh=_normal(g, (rows, cols), 1e-1, rd))
            for k in s["leaves"]:
                s[k].requires_grad_(True)
        return s
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    n = case["tokens"]
    if case["kind"] == "rotary":
        qkv = _normal(g, (n, hq + 2 * hk, d), 1.0, dt)
        f, s["factor"] = _frequencies(case["part"], case["scaling"], case["far"])
        # documents one behind the other, each counted from a place of its own
        start = int(torch.randint(0, case["far"], (1,), generator=g, device=DEVICE)) if n < case["far"] else 0
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], positions=(torch.arange(n, device=DEVICE) + start) % case["far"],
                 frequencies=torch.tensor(f, dtype=torch.float64, device=DEVICE))
        if case["train"]:
            s.update(dq=_normal(g, (n, hq, d), 1e-1, dt), dk=_normal(g, (n, hk, d), 1e-1, dt))
            s["q"], s["k"] = s["q"].requires_grad_(True), s["k"].requires_grad_(True)
        return s
    if "context" in case:
        b, m = case["batch"], case["context"]
        room = m + 64   # a cache has room for more
        s["q"] = _normal(g, (b, n, hq, d), 1.5, dt)
        s["k"], s["v"] = (_normal(g, (b, room, hk, d), 1.0, dt)[:, :m] for _ in range(2))
        return s
    qkv = _normal(g, (n, hq + 2 * hk, d), 1.0, dt)
    ends = [0]
    for length in _lengths(case):
        ends.append(ends[-1] + length)
    # queries and keys come from the rotation, values lie where the linear left them
    s.update(q=(qkv[:, :hq] * 1.5).requires_grad_(True), k=qkv[:, hq:hq + hk].contiguous().requires_grad_(True), v=qkv[:, hq + hk:].requires_grad_(True),
             do=_normal(g, (n, hq, d), 1e-1, dt), ends=ends, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device=DEVICE))
    return s


# ------------------------------------------------------------------------------------------------ the operators
def run(s):
    return {"attention": _attention, "rotary": _rotary, "norms": _norms}[s["kind"]](s)


def _attention(s):
    step = "do" in s
    if own:
        from nanotron_amd.nn import attention

        if not step:
            with torch.no_grad():
                return attention(s["q"], s["k"], s["v"], causal=s["causal"])
        out = attention(s["q"], s["k"], s["v"], cu_seqlens=s["cu_seqlens"], causal=s["causal"])
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"]))
    with torch.no_grad():
        if not step:
            b = max(1, SCORES // (s["heads"] * s["tokens"] * s["context"]))   # sequences at a time
            at = range(0, s["batch"], b)
            return torch.cat([_plain(s["q"][i:i + b], s["k"][i:i + b], s["v"][i:i + b], s["causal"])[0] for i in at]).to(s["q"].dtype)
        outs = [torch.empty_like(s[k], memory_format=torch.contiguous_format) for k in ("q", "q", "k", "v")]
        group = s["heads"] // s["kv_heads"]
        for a, e in zip(s["ends"], s["ends"][1:]):
            if a == e:
                continue
            few = max(1, SCORES // (group * (e - a) ** 2))   # key heads at a time
            for h in range(0, s["kv_heads"], few):
                kv, hs = slice(h, h + few), slice(h * group, (h + few) * group)
                q, k, v, do = (s[n][a:e, w][None] for n, w in (("q", hs), ("k", kv), ("v", kv), ("do", hs)))
                for o, w, t in zip(outs, (hs, hs, kv, kv), _plain(q, k, v, s["causal"], do)):
                    o[a:e, w] = t[0]
        return tuple(outs)


def _plain(q, k, v, causal, do=None):
    """[batch, rows, heads, dim] -> the output, with `do` also the gradients of q, k and v."""
    b, n, hq, d = q.shape
    m, hk = k.shape[1], k.shape[2]
    group, scale = hq // hk, d ** -0.5

    def by_head(t):      # [batch, heads, rows, dim] in fp32
        return t.float().permute(0, 2, 1, 3).contiguous()

    def grouped(t):      # the heads of a group as rows of one matrix
        return by_head(t).view(b, hk, group * n, d)

    def back(t):
        return t.view(b, hq, n, d).permute(0, 2, 1, 3)

    qf, kf, vf = grouped(q), by_head(k), by_head(v)
    x = (qf @ kf.transpose(-1, -2)).mul_(scale)
    if causal and n > 1:
        seen = torch.arange(m, device=q.device) <= torch.arange(m - n, m, device=q.device)[:, None]
        x.view(b, hk, group, n, m).masked_fill_(~seen, -math.inf)
    p = torch.exp_(x.sub_(x.amax(-1, keepdim=True)))
    p /= p.sum(-1, keepdim=True)
    o = p @ vf
    if do is None:
        return (back(o),)
    g = grouped(do)
    dv = p.transpose(-1, -2) @ g
    delta = (g * o).sum(-1, keepdim=True)
    ds = (g @ vf.transpose(-1, -2)).sub_(delta).mul_(p).mul_(scale)
    return back(o), back(ds @ kf), (ds.transpose(-1, -2) @ qf).permute(0, 2, 1, 3), dv.permute(0, 2, 1, 3)


def _rotary(s):
    if own:
        from nanotron_amd.nn import rotary

        call = dict(interleaved=s["interleaved"], scale=s["factor"])
        if not s["train"]:
            with torch.no_grad():
                return rotary(s["q"], s["k"], s["positions"], s["frequencies"], **call)
        q, k = rotary(s["q"], s["k"], s["positions"], s["frequencies"], **call)
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    with torch.no_grad():
        angle = s["positions"].double()[:, None] * s["frequencies"]
        cos, sin = ((t * s["factor"]).float()[:, None] for t in (angle.cos(), angle.sin()))

        def turn(x, sin):
            out, part = torch.empty(x.shape, dtype=x.dtype, device=x.device), s["part"]
            f = x[..., :part].float()
            if s["interleaved"]:
                a, b = f[..., 0::2], f[..., 1::2]
                out[..., 0:part:2], out[..., 1:part:2] = a * cos - b * sin, b * cos + a * sin
            else:
                a, b = f[..., :part // 2], f[..., part // 2:]
                out[..., :part // 2], out[..., part // 2:part] = a * cos - b * sin, b * cos + a * sin
            out[..., part:] = x[..., part:]
            return out

        ahead = turn(s["q"], sin), turn(s["k"], sin)
        return ahead if not s["train"] else (*ahead, turn(s["dq"], -sin), turn(s["dk"], -sin))


def _norms(s):
    if own:
        from nanotron_amd.nn import residual_rms_norm

        call = dict(post_weight=s["post_weight"], gate=s["channel"], residual_scale=s["scale"], eps=EPS)
        if not s["train"]:
            with torch.no_grad():
                return residual_rms_norm(s["x"], s["residual"], s["weight"], **call)
        y, h = residual_rms_norm(s["x"], s["residual"], s["weight"], **call)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), [s[k] for k in s["leaves"]], (s["dy"], s["dh"])))
    with torch.no_grad():
        x, w = s["x"].float(), s["weight"].float()
        p = x
        if s["post"]:
            first = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            u = x * first
            pw = s["post_weight"].float()
            p = u * pw
        gate = s["channel"].float() if s["channel"] is not None else None
        h = s["residual"].float() * s["scale"] + (p if gate is None else gate * p)
        h = h.to(s["residual"].dtype)
        hf = h.float()
        second = 1 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
        n = hf * second
        y = (n * w).to(s["x"].dtype)
        if not s["train"]:
            return y, h
        dy = s["dy"].float()
        a = dy * w
        dh = s["dh"].float() + second * (a - n * (a * n).mean(-1, keepdim=True))
        grads = dict(residual=dh * s["scale"], weight=(dy * n).sum(0))
        if gate is not None:
            grads["channel"] = dh * p if s["gate"] == "element" else (dh * p).sum(0)
        dp = dh if gate is None else dh * gate
        if s["post"]:
            grads["post_weight"] = (dp * u).sum(0)
            c = dp * pw
            dp = first * (c - u * (c * u).mean(-1, keepdim=True))
        grads["x"] = dp
        return (y, h, *[grads[k].to(s[k].dtype) for k in s["leaves"]])


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "rotary": _exact_rotary, "norms": _exact_norms}[case["kind"]](s)


def _exact_attention(s):
    step = "do" in s
    group, scale = s["heads"] // s["kv_heads"], 1 / math.sqrt(s["dim"])

    def head(q, k, v, do):    # one query head of one sequence
        x = torch.mm(q, k.t()) * scale
        if s["causal"]:
            x += torch.full_like(x, -math.inf).triu_(k.shape[0] - q.shape[0] + 1)
        p = torch.softmax(x, -1)
        o = torch.mm(p, v)
        if do is None:
            return o, None, None, None
        dv = torch.mm(p.t(), do)
        dp = torch.mm(do, v.t())
        ds = p.mul_(dp.sub_((do * o).sum(1)[:, None])).mul_(scale)
        return o, torch.mm(ds, k), torch.mm(ds.t(), q), dv

    if not step:
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for b in range(s["batch"]):
            for h in range(s["heads"]):
                out[b, :, h] = head(s["q"][b, :, h].double(), s["k"][b, :, h // group].double(), s["v"][b, :, h // group].double(), None)[0]
        return out
    o, dq, dk, dv = (torch.zeros(s[k].shape, dtype=torch.float64, device=DEVICE) for k in ("q", "q", "k", "v"))
    for a, e in zip(s["ends"], s["ends"][1:]):
        for h in range(s["heads"] if e > a else 0):
            j = h // group
            r = head(*(t.double() for t in (s["q"][a:e, h], s["k"][a:e, j], s["v"][a:e, j], s["do"][a:e, h])))
            o[a:e, h], dq[a:e, h] = r[0], r[1]
            dk[a:e, j] += r[2]
            dv[a:e, j] += r[3]
    return o, dq, dk, dv


def _exact_rotary(s):
    turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device=DEVICE), s["positions"].double()[:, None, None] * s["frequencies"])

    def rotated(x, by):
        x, part = x.double(), s["part"]
        pairs = x[..., :part].unflatten(-1, (part // 2, 2)) if s["interleaved"] else x[..., :part].unflatten(-1, (2, part // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z if s["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.reshape(*x.shape[:-1], part), x[..., part:]], -1)

    ahead = rotated(s["q"], turn), rotated(s["k"], turn)
    return ahead if not s["train"] else (*ahead, rotated(s["dq"], turn.conj()), rotated(s["dk"], turn.conj()))


def _exact_norms(s):
    x, r, w = s["x"].double(), s["residual"].double(), s["weight"].double()
    inner = x
    if s["post"]:
        first = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        inner = x * first * s["post_weight"].double()
    gate = 1.0 if s["channel"] is None else s["channel"].double()
    # the second norm reads h as it is kept
    h = (s["scale"] * r + gate * inner).to(s["residual"].dtype)
    hd = h.double()
    second = (hd.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = hd * second * w
    full = s["scale"] * r + gate * inner
    if not s["train"]:
        return y, full
    dy = s["dy"].double()
    inside = dy * w * second
    dh = s["dh"].double() + inside - hd * second.square() * (inside * hd).mean(-1, keepdim=True)
    found = {"residual": dh * s["scale"], "weight": (dy * hd * second).sum(0)}
    if s["channel"] is not None:
        found["channel"] = dh * inner if s["gate"] == "element" else (dh * inner).sum(0)
    back = dh * gate
    if s["post"]:
        found["post_weight"] = (back * x * first).sum(0)
        back = back * s["post_weight"].double() * first
        back = back - x * first.square() * (back * x).mean(-1, keepdim=True)
    found["x"] = back
    return (y, full, *[found[k] for k in s["leaves"]])


# ------------------------------------------------------------------------------------------------ work
def work(case):
    b = BYTES[case["dtype"]]
    if case["kind"] == "norms":
        n, c, rb, wb = case["rows"] * case["cols"], case["cols"], BYTES[case["rdtype"]], BYTES[case["wdtype"]]
        element, vectors = case["gate"] == "element", 1 + case["post"] + (case["gate"] == "channel")
        once = n * (b + rb + b * element) + vectors * c * wb       # x, the residual, the gate and the weights: what comes in, and each one's gradient
        return {"bytes": (2 if case["train"] else 1) * once + n * (b + rb) * (2 if case["train"] else 1), "flops": (40 if case["train"] else 12) * n}
    hq, hk, d, n = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    if case["kind"] == "rotary":
        times = 2 if case["train"] else 1
        return {"bytes": times * 2 * n * (hq + hk) * d * b + 8 * n + 4 * case["part"], "flops": times * n * (hq + hk) * case["part"] * 3}
    pairs = _pairs(case)
    if "context" in case:
        return {"bytes": case["batch"] * d * b * (2 * n * hq + 2 * case["context"] * hk), "flops": 4 * pairs * hq * d}
    # forward q k^T and p v; backward dp, dv, dq, dk and the scores once more, which no layer keeps
    return {"bytes": 4 * n * (hq + hk) * d * b, "flops": 14 * pairs * hq * d}
