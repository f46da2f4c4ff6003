"""Binding of the operators of include/ntops.h: the host extension that serves the public modules, and the C entry points
themselves for callers that hold device pointers.

There is no fallback: if the library is missing the import fails."""
import ctypes

from nanotron_amd import _native as nt

try:
    from nanotron_amd import _opscall as host
except ImportError as e:
    raise ImportError(f"nanotron_amd/_opscall.so is missing or does not match this torch ({e}): build it first "
                      "(python -m nanotron_amd.build)") from e

_c = ctypes
_vp, _i, _i64, _f, _d = _c.c_void_p, _c.c_int, _c.c_int64, _c.c_float, _c.c_double
ADAMW_BLOCK = 256


class AdamWTensor(ctypes.Structure):
    """`ntops_adamw_tensor` of include/ntops.h."""
    _fields_ = [("param", _vp), ("grad", _vp), ("exp_avg", _vp), ("exp_avg_sq", _vp), ("copy", _vp), ("exp_avg_scale", _vp),
                ("exp_avg_sq_scale", _vp), ("n", _i64)]


class AdamWOptions(ctypes.Structure):
    """`ntops_adamw_options` of include/ntops.h."""
    _fields_ = [("lr", _d), ("beta1", _d), ("beta2", _d), ("eps", _d), ("weight_decay", _d), ("step", _i64), ("param_dtype", _i),
                ("grad_dtype", _i), ("copy_dtype", _i), ("bits", _i), ("seed", _c.c_uint32), ("grad_scale", _vp)]


class LinearCrossEntropyDesc(ctypes.Structure):
    """`ntops_linear_cross_entropy_desc` of include/ntops.h."""
    _fields_ = [("x", _vp), ("weight", _vp), ("labels", _vp), ("tokens", _i64), ("hidden", _i64), ("vocab", _i64), ("x_stride", _i64),
                ("weight_stride", _i64), ("ignore_index", _i64), ("x_dtype", _i), ("mean", _i), ("grad_dtype", _i), ("losses", _vp),
                ("loss", _vp), ("dx", _vp), ("dweight", _vp), ("workspace", _vp)]


class ScaleTensor(ctypes.Structure):
    """`ntops_scale_tensor` of include/ntops.h."""
    _fields_ = [("x", _vp), ("out", _vp), ("n", _i64)]


class RmsNormDesc(ctypes.Structure):
    """`ntops_rms_norm_desc` of include/ntops.h."""
    _fields_ = [("x", _vp), ("residual", _vp), ("gate", _vp), ("weight", _vp), ("post_weight", _vp), ("rows", _i64),
                ("cols", _i64), ("x_stride", _i64), ("residual_stride", _i64), ("gate_stride", _i64), ("x_dtype", _i),
                ("residual_dtype", _i), ("w_dtype", _i), ("gate_kind", _i), ("eps", _f), ("residual_scale", _f), ("y", _vp),
                ("h", _vp), ("first", _vp), ("second", _vp)]


class RmsNormGrads(ctypes.Structure):
    """`ntops_rms_norm_grads` of include/ntops.h."""
    _fields_ = [("dy", _vp), ("dh", _vp), ("dy_stride", _i64), ("dh_stride", _i64), ("dx", _vp), ("dresidual", _vp),
                ("dgate", _vp), ("dweight", _vp), ("dpost_weight", _vp), ("scratch", _vp)]


class RotaryDesc(ctypes.Structure):
    """`ntops_rotary_desc` of include/ntops.h."""
    _fields_ = [("q", _vp), ("k", _vp), ("q_out", _vp), ("k_out", _vp), ("tokens", _i64), ("q_stride", _i64), ("q_head", _i64),
                ("k_stride", _i64), ("k_head", _i64), ("heads", _i), ("kv_heads", _i), ("head_dim", _i), ("pairs", _i),
                ("dtype", _i), ("positions", _vp), ("position_count", _i64), ("position_bits", _i), ("frequencies", _vp),
                ("interleaved", _i), ("inverse", _i), ("scale", _f)]


class AttentionDesc(ctypes.Structure):
    """`ntops_attention_desc` of include/ntops.h."""
    _fields_ = [("q", _vp), ("k", _vp), ("v", _vp), ("q_stride", _i64), ("k_stride", _i64), ("v_stride", _i64),
                ("q_head", _i64), ("k_head", _i64), ("v_head", _i64), ("q_batch", _i64), ("k_batch", _i64), ("v_batch", _i64),
                ("cu_q", _vp), ("cu_k", _vp), ("sequences", _i64), ("q_rows", _i64), ("k_rows", _i64), ("heads", _i),
                ("kv_heads", _i), ("head_dim", _i), ("dtype", _i), ("causal", _i), ("scale", _f), ("out", _vp), ("out_low", _vp), ("lse", _vp),
                ("workspace", _vp), ("plan", _vp), ("dout", _vp), ("do_stride", _i64), ("do_head", _i64), ("do_batch", _i64), ("dq", _vp),
                ("dk", _vp), ("dv", _vp)]


SIGNATURES = {
    "ntops_layer_norm_forward": (_i, [_vp, _i, _i64, _i64, _i64, _vp, _vp, _i, _f, _vp, _vp, _vp, _vp]),
    "ntops_layer_norm_scratch": (_i64, [_i, _i64, _i64]),
    "ntops_layer_norm_backward": (_i, [_vp, _i64, _vp, _i, _i64, _i64, _i64, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ntops_adamw": (_i, [_c.POINTER(AdamWTensor), _i, _c.POINTER(AdamWOptions), _vp]),
    "ntops_adamw_check": (_i, [_c.POINTER(AdamWTensor), _i, _c.POINTER(AdamWOptions)]),
    "ntops_adamw_unpack": (_i, [_vp, _vp, _i64, _vp, _vp]),
    "ntops_linear_cross_entropy_piece": (_i64, [_i64]),
    "ntops_linear_cross_entropy_workspace": (_i64, [_c.POINTER(LinearCrossEntropyDesc)]),
    "ntops_linear_cross_entropy": (_i, [_c.POINTER(LinearCrossEntropyDesc), _vp]),
    "ntops_rms_norm_forward": (_i, [_c.POINTER(RmsNormDesc), _vp]),
    "ntops_rms_norm_scratch": (_i64, [_c.POINTER(RmsNormDesc)]),
    "ntops_rms_norm_backward": (_i, [_c.POINTER(RmsNormDesc), _c.POINTER(RmsNormGrads), _vp]),
    "ntops_rotary": (_i, [_c.POINTER(RotaryDesc), _vp]),
    "ntops_attention_workspace": (_i64, [_c.POINTER(AttentionDesc), _i]),
    "ntops_attention_plan": (_i64, [_c.POINTER(AttentionDesc)]),
    "ntops_attention_forward": (_i, [_c.POINTER(AttentionDesc), _vp]),
    "ntops_attention_backward": (_i, [_c.POINTER(AttentionDesc), _vp]),
    "ntops_scale": (_i, [_c.POINTER(ScaleTensor), _i, _i, _vp, _i, _vp]),
}
for _name, (_res, _args) in SIGNATURES.items():
    _fn = getattr(nt.lib, _name)  # AttributeError here = library / header mismatch
    _fn.restype = _res
    _fn.argtypes = _args
lib = nt.lib
