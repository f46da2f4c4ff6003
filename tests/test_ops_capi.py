"""CPU-side checks of the operators' C ABI: every declared symbol is exported and bound, struct layouts agree, argument
errors come back as codes before any launch, and the public functions refuse what they cannot serve."""
import ctypes
import os
import re

import pytest
import torch

from nanotron_amd import _native as nt
from nanotron_amd import _ops
from nanotron_amd.nn import LayerNorm, layer_norm, linear_cross_entropy
from nanotron_amd.optim import AdamW, adamw_step

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ntops.h")
P, Q, R = 0x10000, 0x20000000, 0x40000000   # never dereferenced: validation fails first
NULL, ENUM, SIZE, ALIGN, UNSUPPORTED, ALIAS = -1, -2, -3, -4, -5, -7


def source():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_library_exports_every_declared_symbol():
    names = sorted(set(re.findall(r"\b(ntops_[a-z0-9_]+)\s*\(", source())))
    assert sorted(_ops.SIGNATURES) == names
    for n in names:
        assert hasattr(_ops.lib, n)
    assert int(re.search(r"#define NTOPS_ADAMW_BLOCK (\d+)", open(HEADER).read()).group(1)) == _ops.ADAMW_BLOCK


@pytest.mark.parametrize("name,struct", [("ntops_adamw_tensor", _ops.AdamWTensor), ("ntops_adamw_options", _ops.AdamWOptions),
                                         ("ntops_linear_cross_entropy_desc", _ops.LinearCrossEntropyDesc), ("ntops_scale_tensor", _ops.ScaleTensor)])
def test_struct_fields_match_header(name, struct):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), source(), flags=re.S).group(1)
    fields = []
    for line in body.split(";"):
        if line.strip():
            fields += [re.split(r"[\s*]+", part.strip())[-1] for part in line.split(",")]
    assert fields == [f[0] for f in struct._fields_]


def test_layer_norm_argument_errors():
    f, b = _ops.lib.ntops_layer_norm_forward, _ops.lib.ntops_layer_norm_backward
    assert f(None, 2, 4, 8, 8, P, P, 0, 1e-5, Q, None, None, None) == NULL
    assert f(P, 2, 4, 8, 8, P, P, 0, 1e-5, None, None, None, None) == NULL
    assert f(P, 2, 4, 8, 8, P, P, 0, 1e-5, Q, R, None, None) == NULL
    assert f(P, 7, 4, 8, 8, P, P, 0, 1e-5, Q, None, None, None) == ENUM
    assert f(P, 2, 4, 8, 8, P, P, 1, 1e-5, Q, None, None, None) == ENUM      # fp16 weights beside bf16 rows
    assert f(P, 2, 0, 8, 8, P, P, 0, 1e-5, Q, None, None, None) == SIZE
    assert f(P, 2, 4, 8, 7, P, P, 0, 1e-5, Q, None, None, None) == SIZE
    assert f(P, 2, 4, 32769, 32769, P, P, 0, 1e-5, Q, None, None, None) == UNSUPPORTED
    assert f(P, 0, 4, 16385, 16385, P, P, 0, 1e-5, Q, None, None, None) == UNSUPPORTED
    assert f(P + 1, 2, 4, 8, 8, P, P, 0, 1e-5, Q, None, None, None) == ALIGN
    assert f(P, 2, 4, 8, 8, P + 2, P, 0, 1e-5, Q, None, None, None) == ALIGN
    assert f(P, 2, 4, 8, 8, Q, Q, 0, 1e-5, P + 16, None, None, None) == ALIAS
    assert b(None, 8, P, 2, 4, 8, 8, P, 0, P, P, Q, Q, Q, R, None) == NULL
    assert b(P, 8, P, 2, 4, 8, 8, P, 0, P, P, None, None, None, R, None) == NULL
    assert b(P, 8, P, 2, 4, 8, 8, P, 0, P, P, Q, Q, Q, None, None) == NULL
    assert b(P, 4, P, 2, 4, 8, 8, P, 0, P, P, Q, Q, Q, R, None) == SIZE
    assert b(P, 8, P, 2, 4, 8, 8, P, 0, P, P, Q, Q, Q, R + 4, None) == ALIGN
    assert b(P, 8, Q, 2, 4, 8, 8, Q, 0, Q, Q, P, None, None, None, None) == ALIAS
    assert _ops.lib.ntops_layer_norm_scratch(2, 0, 8) == 0
    assert _ops.lib.ntops_layer_norm_scratch(2, 1, 8) == 64


def options(**kw):
    o = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=1, param_dtype=0, grad_dtype=0, copy_dtype=0, bits=32, seed=0, grad_scale=None)
    return _ops.AdamWOptions(**{**o, **kw})


def tensors(**kw):
    t = dict(param=P, grad=Q, exp_avg=R, exp_avg_sq=R + 4096, copy=None, exp_avg_scale=None, exp_avg_sq_scale=None, n=16)
    return (_ops.AdamWTensor * 1)(_ops.AdamWTensor(**{**t, **kw}))


def test_adamw_argument_errors():
    f = _ops.lib.ntops_adamw
    assert f(tensors(), 1, None, None) == NULL
    assert f(None, 1, options(), None) == NULL
    for k in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert f(tensors(**{k: None}), 1, options(), None) == NULL
        assert f(tensors(**{k: P + 0x800001}), 1, options(), None) == ALIGN
    assert f(tensors(), 1, options(bits=8), None) == NULL          # no scales
    assert f(tensors(), 1, options(bits=16), None) == ENUM
    assert f(tensors(), 1, options(grad_dtype=5), None) == ENUM
    assert f(tensors(copy=P + 0x100000), 1, options(copy_dtype=-1), None) == ENUM
    assert f(tensors(), 1, options(step=0), None) == SIZE
    assert f(tensors(n=-1), 1, options(), None) == SIZE
    assert f(tensors(), 1, options(beta2=1.0), None) == UNSUPPORTED
    assert f(tensors(), 1, options(eps=float("nan")), None) == UNSUPPORTED
    assert f(tensors(grad=P), 1, options(), None) == ALIAS
    assert f(tensors(copy=R), 1, options(), None) == ALIAS
    assert f(tensors(n=0, param=None), 1, options(), None) == 0    # nothing to do, nothing launched
    assert f(None, 0, options(), None) == 0
    g = _ops.lib.ntops_adamw_unpack
    assert g(None, P, 4, Q, None) == NULL and g(P, P, 0, Q, None) == SIZE and g(P, R, 64, P + 16, None) == ALIAS


def desc(**kw):
    d = dict(x=P, weight=0x1000000, labels=0x2000000, tokens=16, hidden=64, vocab=1000, x_stride=64, weight_stride=64, ignore_index=-100,
             x_dtype=nt.BF16, mean=1, grad_dtype=nt.BF16, losses=0x3000000, loss=0x3100000, dx=0x4000000, dweight=0x5000000, workspace=0x10000000)
    return _ops.LinearCrossEntropyDesc(**{**d, **kw})


def test_linear_cross_entropy_argument_errors():
    f = _ops.lib.ntops_linear_cross_entropy
    assert f(None, None) == NULL
    for k in ("x", "weight", "labels", "losses", "workspace"):
        assert f(desc(**{k: None}), None) == NULL
    assert f(desc(x_dtype=nt.F32), None) == ENUM
    assert f(desc(grad_dtype=nt.F16), None) == ENUM
    for k in ("tokens", "hidden", "vocab"):
        assert f(desc(**{k: 0}), None) == SIZE
    assert f(desc(x_stride=63), None) == SIZE and f(desc(vocab=1 << 23), None) == SIZE
    piece = _ops.lib.ntops_linear_cross_entropy_piece(128000)
    assert piece == 8192
    assert f(desc(vocab=128000, tokens=piece + 1), None) == UNSUPPORTED
    assert f(desc(x=P + 1), None) == ALIGN and f(desc(workspace=0x10000010), None) == ALIGN and f(desc(dx=0x4000004), None) == ALIGN
    assert f(desc(dx=P), None) == ALIAS and f(desc(loss=0x3000000), None) == ALIAS and f(desc(workspace=0x5000000), None) == ALIAS
    size = _ops.lib.ntops_linear_cross_entropy_workspace
    assert size(desc(tokens=0)) == 0
    # two bytes a logit, bounded
    assert size(desc(tokens=64, vocab=128000)) < 2 * 64 * 128000 * 1.3
    assert size(desc(tokens=1 << 16, vocab=128000, grad_dtype=nt.F32)) < (1 << 31) * 1.2


def test_scale_argument_errors():
    def f(x=P, out=Q, n=4, x_dtype=0, factor=R, out_dtype=0, count=1):
        return _ops.lib.ntops_scale((_ops.ScaleTensor * 1)(_ops.ScaleTensor(x, out, n)), count, x_dtype, factor, out_dtype, None)

    assert f(x=None) == NULL and f(out=None) == NULL and f(factor=None) == NULL and _ops.lib.ntops_scale(None, 1, 0, R, 0, None) == NULL
    assert f(x_dtype=3) == ENUM and f(out_dtype=-1) == ENUM and f(n=0) == SIZE and f(count=-1) == SIZE
    assert f(out=P, out_dtype=2) == ALIAS and f(x=P + 2) == ALIGN and f(count=0) == 0


def test_public_functions_refuse_host_tensors():
    x = torch.ones(3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        linear_cross_entropy(x, x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        adamw_step([x], [x], [x], [x], lr=1e-3, step=1)
    adamw_step([], [], [], [], lr=1e-3, step=1)


def test_constructors_refuse():
    with pytest.raises(ValueError, match="last dimension"):
        LayerNorm((4, 8))
    with pytest.raises(ValueError, match="last dimension"):
        LayerNorm(8)(torch.ones(3, 7))
    p = torch.nn.Parameter(torch.ones(4))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(ValueError, match="copies"):
        AdamW([dict(params=[p], copies=[None, None])])
    assert ctypes.sizeof(_ops.AdamWTensor) == 64


def test_adamw_addresses():
    for k in ("param", "grad", "exp_avg", "exp_avg_sq", "copy"):
        assert _ops.lib.ntops_adamw(tensors(**{k: 1 << 48}), 1, options(copy_dtype=nt.BF16), None) == UNSUPPORTED


def test_linear_cross_entropy_takes_rows_far_apart():
    """Strides are bounded by what can be addressed alone; rows further apart than tiles reach are copied, which the workspace says."""
    size = _ops.lib.ntops_linear_cross_entropy_workspace
    near, far = 1 << 22, (1 << 22) + 8
    for g in (dict(), dict(dx=None, dweight=None)):
        base = size(desc(x_stride=near, weight_stride=near, **g))
        assert base > 0
        assert size(desc(x_stride=far, weight_stride=near, **g)) == base + (0 if not g else 16 * 64 * 2)      # (with gradients x is gathered anyway)
        assert size(desc(x_stride=near, weight_stride=far, **g)) == base + 1000 * 64 * 2
    assert _ops.lib.ntops_linear_cross_entropy(desc(x_stride=(1 << 46) // 16 + 8), None) == SIZE
    assert _ops.lib.ntops_linear_cross_entropy(desc(weight_stride=(1 << 46) // 1000 + 8), None) == SIZE


def test_adamw_check_says_what_a_step_would():
    f, g = _ops.lib.ntops_adamw_check, _ops.lib.ntops_adamw
    for t, o in ((tensors(), options(bits=8)), (tensors(), options(step=0)), (tensors(grad=P), options()), (tensors(param=P + 0x800001), options()),
                 (tensors(exp_avg=1 << 48), options()), (tensors(n=0, param=None), options())):
        assert f(t, 1, o) == g(t, 1, o, None)
    assert f(tensors(), 1, options()) == 0 and f(None, 1, options()) == NULL and f(tensors(), 1, None) == NULL


def test_adamw_takes_the_state_of_torch():
    p = [torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(3, dtype=torch.bfloat16))]
    theirs = torch.optim.AdamW(p, lr=0.25)
    for q in p:
        q.grad = torch.ones_like(q)
    theirs.step()
    ours = AdamW(p, state_bits=8, seed=5)
    ours.load_state_dict(theirs.state_dict())
    group = ours.param_groups[0]
    # (its moments are 32-bit ones)
    assert group["lr"] == 0.25 and group["state_bits"] == 32 and group["seed"] == 5 and group["copies"] is None
    for q in p:
        state = ours.state[q]
        assert type(state["step"]) is int and state["step"] == 1
        assert state["exp_avg"].dtype == state["exp_avg_sq"].dtype == torch.float32
        assert torch.equal(state["exp_avg"], theirs.state[q]["exp_avg"].float())
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError, match=next(iter(kw))):
            AdamW(p).load_state_dict(torch.optim.AdamW(p, **kw).state_dict())
    with pytest.raises(ValueError, match="decoupled"):
        AdamW(p).load_state_dict(torch.optim.Adam(p, weight_decay=0.1).state_dict())
    AdamW(p).load_state_dict(torch.optim.Adam(p).state_dict())


def test_a_refused_group_is_not_added():
    p, q = (torch.nn.Parameter(torch.ones(4)) for _ in range(2))
    o = AdamW([p])
    for kw in (dict(copies=[None, None]), dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError, match=next(iter(kw))):
            o.add_param_group(dict(params=[q], **kw))
        assert [g["params"] for g in o.param_groups] == [[p]]
        with pytest.raises(ValueError, match=next(iter(kw))):
            AdamW([dict(params=[q], **kw)])
    o.add_param_group(dict(params=[q], copies=[None], state_bits=8))
    assert len(o.param_groups) == 2


def test_workspace_of_many_tokens_of_few_labels():
    """Beside the logits, the sums of dx in fp32, at most 2 GiB of each, with 8 bytes for 128 logits and 24 for a token on top."""
    size = _ops.lib.ntops_linear_cross_entropy_workspace
    for tokens, hidden, vocab in ((1 << 18, 8192, 1000), (1 << 16, 8192, 8000), (1 << 17, 16384, 500), (70000, 8200, 300), (4096, 4096, 128000), (3000, 65536, 1000)):
        logits = min(1 << 31, 2 * tokens * (vocab + 63))
        dx = min(1 << 31, 4 * (tokens + 255) * hidden)
        # fewer rows than the chip has room for are cut into runs of the vocabulary: 1024 tiles of 256 x 256 at most
        dx = max(dx, 1024 << 18)
        d = desc(tokens=tokens, hidden=hidden, vocab=vocab, x_stride=hidden, weight_stride=hidden)
        assert size(d) <= logits * 1.04 + dx + 2 * tokens * hidden + 24 * tokens + (1 << 16), (tokens, hidden, vocab)
        assert size(desc(tokens=tokens, hidden=hidden, vocab=vocab, x_stride=hidden, weight_stride=hidden, dx=None)) <= logits * 1.04 + 2 * tokens * hidden + 24 * tokens + (1 << 16)


def test_a_group_of_wrong_types_is_not_added():
    o = AdamW([torch.nn.Parameter(torch.ones(4))])
    for kw in (dict(copies=iter([None])), dict(lr="high"), dict(betas=0.9)):
        with pytest.raises(TypeError):
            o.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(4))], **kw))
        assert len(o.param_groups) == 1
