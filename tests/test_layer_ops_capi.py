"""CPU-side checks of the C ABI of attention, rotary positions and the norms around a block: struct layouts agree with the header, argument errors come
back as codes before any launch, the public functions refuse what they cannot serve, and frequencies are what their formulas say."""
import math
import os
import re

import pytest
import torch

from nanotron_amd import _native as nt
from nanotron_amd import _ops
from nanotron_amd.nn import RMSNorm, RotaryEmbedding, attention, residual_rms_norm, rms_norm, rotary, rotary_frequencies

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ntops.h")
NULL, ENUM, SIZE, ALIGN, UNSUPPORTED, ALIAS = -1, -2, -3, -4, -5, -7
KINDS = {"int64_t": _ops._i64, "int": _ops._i, "float": _ops._f}


@pytest.mark.parametrize("name,struct", [("ntops_rms_norm_desc", _ops.RmsNormDesc), ("ntops_rms_norm_grads", _ops.RmsNormGrads), ("ntops_rotary_desc", _ops.RotaryDesc),
                                         ("ntops_attention_desc", _ops.AttentionDesc)])
def test_struct_fields_match_header(name, struct):
    source = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), source, flags=re.S).group(1)
    fields = []
    for line in filter(None, (x.strip() for x in body.split(";"))):
        kind = _ops._vp if "*" in line else KINDS[line.split()[0]]
        fields += [(re.split(r"[\s*]+", part.strip())[-1], kind) for part in line.split(",")]
    assert fields == [tuple(f) for f in struct._fields_]


def norms(**kw):
    d = dict(x=0x100000, residual=0x200000, gate=None, weight=0x300000, post_weight=None, rows=4, cols=64, x_stride=64, residual_stride=64, gate_stride=0, x_dtype=nt.BF16,
             residual_dtype=nt.F32, w_dtype=nt.F32, gate_kind=0, eps=1e-6, residual_scale=1.0, y=0x400000, h=0x500000, first=None, second=None)
    return _ops.RmsNormDesc(**{**d, **kw})


def test_rms_norm_argument_errors():
    f = _ops.lib.ntops_rms_norm_forward
    assert f(None, None) == NULL
    for kw in (dict(x=None), dict(y=None), dict(h=None), dict(residual=None), dict(gate_kind=1), dict(gate_kind=2, gate_stride=64), dict(residual=None, h=None, post_weight=0x600000),
               dict(first=0x700000), dict(post_weight=0x600000, second=0x700000)):
        assert f(norms(**kw), None) == NULL, kw
    for kw in (dict(x_dtype=5), dict(residual_dtype=nt.F16), dict(w_dtype=nt.F16), dict(gate_kind=3), dict(residual=None, h=None)):
        assert f(norms(**kw), None) == ENUM, kw
    for kw in (dict(rows=0), dict(cols=0), dict(x_stride=63), dict(residual_stride=63), dict(gate=0x600000, gate_kind=2, gate_stride=63)):
        assert f(norms(**kw), None) == SIZE, kw
    for kw in (dict(cols=16385, x_stride=16385, residual_stride=16385), dict(x_dtype=nt.F32, cols=8193, x_stride=8193, residual_stride=8193), dict(eps=-1.0), dict(eps=math.nan),
               dict(residual_scale=math.nan)):
        assert f(norms(**kw), None) == UNSUPPORTED, kw
    for kw in (dict(x=0x100001), dict(residual=0x200002), dict(weight=0x300002), dict(y=0x400001), dict(h=0x500002)):
        assert f(norms(**kw), None) == ALIGN, kw
    for kw in (dict(y=0x100010), dict(h=0x200010), dict(y=0x500010), dict(h=0x300010)):
        assert f(norms(**kw), None) == ALIAS, kw
    assert _ops.lib.ntops_rms_norm_scratch(norms()) == 64 * 4 and _ops.lib.ntops_rms_norm_scratch(norms(rows=0)) == 0
    assert _ops.lib.ntops_rms_norm_scratch(norms(post_weight=0x600000)) == 3 * 64 * 4

    def b(desc=None, **kw):
        g = dict(dy=0x800000, dh=0x900000, dy_stride=64, dh_stride=64, dx=0xa00000, dresidual=0xb00000, dgate=None, dweight=0xc00000, dpost_weight=None, scratch=0xd00000)
        return _ops.lib.ntops_rms_norm_backward(norms(second=0x700000, y=None, **(desc or {})), _ops.RmsNormGrads(**{**g, **kw}), None)

    assert b(dy=None, dh=None) == NULL and b(scratch=None) == NULL and b(dgate=0xe00000) == NULL and b(dpost_weight=0xe00000) == NULL
    assert b(dict(h=None)) == NULL and b(dict(weight=None)) == NULL and b(dx=None, dresidual=None, dweight=None) == NULL
    assert b(dict(post_weight=0x600000)) == NULL          # without the 1 / rms of x
    assert b(dict(h=None, residual=None), dh=None, dresidual=None) == ENUM
    assert b(dy_stride=63) == SIZE and b(dh_stride=3) == SIZE
    assert b(dy=0x800001) == ALIGN and b(scratch=0xd00004) == ALIGN and b(dresidual=0xb00002) == ALIGN
    assert b(dx=0x800000) == ALIAS and b(dresidual=0xa00010) == ALIAS and b(dweight=0x300000) == ALIAS and b(scratch=0xb00000) == ALIAS


def turns(**kw):
    d = dict(q=0x100000, k=0x200000, q_out=0x300000, k_out=0x400000, tokens=4, q_stride=256, q_head=64, k_stride=128, k_head=64, heads=4, kv_heads=2, head_dim=64, pairs=32,
             dtype=nt.BF16, positions=0x500000, position_count=4, position_bits=64, frequencies=0x600000, interleaved=0, inverse=0, scale=1.0)
    return _ops.RotaryDesc(**{**d, **kw})


def test_rotary_argument_errors():
    f = _ops.lib.ntops_rotary
    assert f(None, None) == NULL
    for kw in (dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(positions=None), dict(frequencies=None), dict(heads=-1)):
        assert f(turns(**kw), None) == NULL, kw
    for kw in (dict(dtype=3), dict(position_bits=16)):
        assert f(turns(**kw), None) == ENUM, kw
    for kw in (dict(tokens=0), dict(heads=0, kv_heads=0), dict(heads=16384), dict(head_dim=0), dict(pairs=0), dict(pairs=33), dict(position_count=0), dict(q_stride=-1)):
        assert f(turns(**kw), None) == SIZE, kw
    assert f(turns(head_dim=2056, q_head=2056), None) == UNSUPPORTED and f(turns(scale=math.nan), None) == UNSUPPORTED
    for kw in (dict(q=0x100001), dict(k_out=0x400001), dict(positions=0x500004), dict(frequencies=0x600004)):
        assert f(turns(**kw), None) == ALIGN, kw
    for kw in (dict(q_out=0x100000), dict(q_out=0x200010), dict(k_out=0x300010), dict(k_out=0x600000)):
        assert f(turns(**kw), None) == ALIAS, kw


def attend(**kw):
    d = dict(q=0x1000000, k=0x2000000, v=0x3000000, q_stride=512, k_stride=128, v_stride=128, q_head=64, k_head=64, v_head=64, q_batch=0, k_batch=0, v_batch=0, cu_q=None,
             cu_k=None, sequences=1, q_rows=100, k_rows=100, heads=8, kv_heads=2, head_dim=64, dtype=nt.BF16, causal=1, scale=0.125, out=0x4000000, lse=None, workspace=0x5000000,
             dout=None, do_stride=512, do_head=64, do_batch=0, dq=None, dk=None, dv=None)
    return _ops.AttentionDesc(**{**d, **kw})


def test_attention_argument_errors():
    f, b = _ops.lib.ntops_attention_forward, _ops.lib.ntops_attention_backward
    assert f(None, None) == NULL and b(None, None) == NULL
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(workspace=None), dict(cu_q=0x6000000), dict(cu_k=0x6000000)):
        assert f(attend(**kw), None) == NULL, kw
    for kw in (dict(dtype=nt.F32), dict(dtype=7)):
        assert f(attend(**kw), None) == ENUM, kw
    for kw in (dict(heads=0), dict(kv_heads=3), dict(head_dim=4), dict(sequences=0), dict(sequences=3), dict(q_rows=0), dict(q_rows=1 << 25), dict(k_rows=-1), dict(q_stride=12),
               dict(k_stride=-8), dict(v_stride=(1 << 24) + 8), dict(k_head=4), dict(q_batch=-8)):
        assert f(attend(**kw), None) == SIZE, kw
    for kw in (dict(head_dim=136), dict(head_dim=60), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)):
        assert f(attend(**kw), None) == UNSUPPORTED, kw
    for kw in (dict(q=0x1000008), dict(v=0x3000002), dict(out=0x4000008), dict(workspace=0x5000080), dict(lse=0x6000002)):
        assert f(attend(**kw), None) == ALIGN, kw
    for kw in (dict(out=0x1000100), dict(out=0x3000100), dict(workspace=0x4000100), dict(lse=0x4000100)):
        assert f(attend(**kw), None) == ALIAS, kw
    grad = dict(dout=0x6000000, lse=0x7000000, dq=0x8000000, dk=0x9000000, dv=0xa000000)
    for kw in (dict(dout=None), dict(lse=None), dict(dq=None, dk=None, dv=None)):
        assert b(attend(**{**grad, **kw}), None) == NULL, kw
    for kw in (dict(dq=0x1000000), dict(dk=0x6000100), dict(dv=0x9000100), dict(dq=0x4000000), dict(workspace=0xa000000)):
        assert b(attend(**{**grad, **kw}), None) == ALIAS, kw
    assert b(attend(**{**grad, "do_stride": 4}), None) == SIZE


def test_attention_workspaces():
    size = _ops.lib.ntops_attention_workspace
    assert size(attend(dtype=0), 0) == 0 and size(attend(), 0) >= 256
    # delta, 4 bytes a query and head, and a task of 32 bytes for every 128 rows and sequence
    assert size(attend(q_rows=1 << 20, k_rows=1 << 20), 1) < (1 << 20) * 8 * 4 + 1024
    packed = dict(cu_q=0x6000000, cu_k=0x6000000, sequences=500)
    assert size(attend(q_rows=1 << 20, k_rows=1 << 20, **packed), 1) < (1 << 20) * 8 * 4 + 2 * 32 * (8192 + 502) + 2048
    # no keys at all: nothing is divided by their tiles
    for kw in (dict(), packed):
        assert size(attend(k_rows=0, k=None, v=None, q_rows=500, **kw), 1) > 0 and size(attend(k_rows=0, q_rows=500, **kw), 0) > 0
    plan = _ops.lib.ntops_attention_plan
    assert plan(attend()) == 0 and plan(attend(q_rows=1 << 20, k_rows=1 << 20, **packed)) < 2 * 32 * (8192 + 502) + 1024
    assert size(attend(q_rows=1 << 20, k_rows=1 << 20, plan=0x7000000, **packed), 1) < size(attend(q_rows=1 << 20, k_rows=1 << 20, **packed), 1)
    # partial results where there are few queries: never more than the chip has room for
    assert size(attend(q_rows=1, k_rows=1 << 20), 0) < 1 << 22


def test_public_functions_refuse_host_tensors():
    x = torch.ones(3, 8)
    h = torch.ones(3, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        residual_rms_norm(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        rotary(h, h, torch.arange(3), rotary_frequencies(8)[0])
    with pytest.raises(ValueError, match="CUDA"):
        attention(h, h, h)


def test_constructors_refuse():
    with pytest.raises(ValueError, match="last dimension"):
        RMSNorm((4, 8))
    with pytest.raises(ValueError, match="last dimension"):
        RMSNorm(8)(torch.ones(3, 7))
    with pytest.raises(ValueError, match="rotary_dim"):
        RotaryEmbedding(64, rotary_dim=66)
    with pytest.raises(ValueError, match="64"):
        RotaryEmbedding(64)(torch.ones(3, 2, 32), None, torch.arange(3))


def test_frequencies():
    f, s = rotary_frequencies(64, 10000.0)
    assert s == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary_frequencies(64, scaling=dict(kind="linear", factor=4.0))[0], f / 4)
    b = rotary_frequencies(64, scaling=dict(kind="base", factor=8.0))[0]
    assert b[0] == 1.0 and abs(b[-1].item() / f[-1].item() * 8 - 1) < 1e-12      # the slowest pair turns as slowly as under "linear"
    w = rotary_frequencies(64, scaling=dict(kind="wavelength", factor=8.0, original=4096, low=1.0, high=4.0))[0]
    for i in range(32):
        wavelength = 2 * math.pi / f[i].item()
        if wavelength < 4096 / 4:
            want = f[i].item()
        elif wavelength > 4096:
            want = f[i].item() / 8
        else:
            t = (4096 / wavelength - 1) / 3
            want = (1 - t) * f[i].item() / 8 + t * f[i].item()
        assert abs(w[i].item() / want - 1) < 1e-12
    y, s = rotary_frequencies(64, scaling=dict(kind="yarn", factor=8.0, original=4096))
    assert s == 0.1 * math.log(8.0) + 1
    turns_ = [4096 * f[i].item() / (2 * math.pi) for i in range(32)]
    lo = max(i for i in range(32) if turns_[i] >= 32)
    hi = min(i for i in range(32) if turns_[i] <= 1)
    assert torch.equal(y[:lo + 1], f[:lo + 1]) and torch.allclose(y[hi:], f[hi:] / 8, rtol=1e-14)
    assert all(f[i] / 8 <= y[i] <= f[i] for i in range(32))
    assert rotary_frequencies(64, scaling=dict(kind="yarn", factor=8.0, original=4096, scale=1.0))[1] == 1.0
    for kw in (dict(kind="other"), dict(kind="linear"), dict(kind="yarn", factor=2.0), dict(kind="linear", factor=2.0, original=4), dict(kind="linear", factor=-1.0),
               dict(kind="wavelength", factor=2.0, original=100, low=4.0, high=1.0), dict(factor=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling=kw)
    for dim in (0, 7, -2):
        with pytest.raises(ValueError):
            rotary_frequencies(dim)
    with pytest.raises(ValueError):
        rotary_frequencies(64, base=1.0)
