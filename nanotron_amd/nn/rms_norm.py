from typing import Optional, Tuple

import torch
from torch import nn

from nanotron_amd import _ops


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Root-mean-square normalisation over the last dimension: `x / sqrt(mean(x**2) + eps) * weight`.

    x: float32, float16 or bfloat16, any number of dimensions; the result has its type.  weight ([x.shape[-1]], optional) is
    float32 or of the type of x.  Arithmetic is fp32.  Up to 16384 columns of a 16-bit x, 8192 of float32.  ValueError / TypeError for
    what does not fit; differentiable once."""
    return _ops.host.rms_norm(x, None, weight, None, None, eps, 1.0)[0]


def residual_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, *, post_weight: Optional[torch.Tensor] = None,
                      gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """What stands between two blocks of a residual stream, in one pass each way.  Returns (y, h):

        h = residual_scale * residual + gate * p        p = rms_norm(x, post_weight), or x without a post_weight
        y = rms_norm(h, weight)

    x is what a block hands on, residual the stream it read from, h the stream behind it and y what the next block reads.

    x [..., columns]: float32, float16 or bfloat16, and y has its type; residual (the shape of x): float32 or of the type of
    x, and so is h.  y is made of h as it was rounded.  gate: one value a channel ([columns]), or one an element (the shape and type of x).  weight,
    post_weight and a channel's gate are optional, float32 or of the type of x, of one type.  Arithmetic is fp32; the gradients of
    weights and of a channel's gate are summed in fp32 within a workgroup and in 64 bits over them, in an order that depends on the
    sizes alone, so gradients repeat bit for bit.  Rows that are dense in themselves (a slice of a wider 2-D tensor) are read where they
    are.  Up to 16384 columns of a 16-bit x, 8192 of float32 (backward with a post_weight or a gate takes 2.5 times as long an element beyond 8192 columns of a 16-bit
    x).  ValueError / TypeError for what does not fit; differentiable once."""
    y, h = _ops.host.rms_norm(x, residual, weight, post_weight, gate, eps, residual_scale)
    return y, h


class RMSNorm(nn.Module):
    """`rms_norm` as a module, with the constructor of torch.nn.RMSNorm for one normalised dimension, but for `eps`, a number here (there None by
    default, the epsilon of the type).  Called with a residual as well, it is `residual_rms_norm` and returns (y, h); `post_norm` and `gate` then say whether the block's output has a norm of its own
    (`post_weight`) and a learned gate for each channel (`gate`, at `gate_init`).  `dtype` is that of the weights, which may stay
    float32 beside 16-bit activations."""

    def __init__(self, normalized_shape: int, eps: float = 1e-6, elementwise_affine: bool = True, device: Optional[torch.device] = None,
                 dtype: Optional[torch.dtype] = None, *, post_norm: bool = False, gate: bool = False, gate_init: float = 1.0, residual_scale: float = 1.0):
        super().__init__()
        if not isinstance(normalized_shape, int):
            if len(normalized_shape) != 1:
                raise ValueError(f"RMSNorm normalises the last dimension, got normalized_shape={normalized_shape}")
            normalized_shape = normalized_shape[0]
        self.normalized_shape, self.eps, self.residual_scale = (normalized_shape,), eps, residual_scale
        made = dict(device=device, dtype=dtype)
        self.weight = nn.Parameter(torch.ones(normalized_shape, **made)) if elementwise_affine else None
        self.post_weight = nn.Parameter(torch.ones(normalized_shape, **made)) if post_norm else None
        self.gate = nn.Parameter(torch.full((normalized_shape,), gate_init, **made)) if gate else None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"the last dimension of x must be {self.normalized_shape[0]}, got shape {tuple(x.shape)}")
        if residual is None:
            if self.post_weight is not None or self.gate is not None:
                raise ValueError("a norm behind the block and a gate go with a residual: RMSNorm(x, residual)")
            return rms_norm(x, self.weight, self.eps)
        return residual_rms_norm(x, residual, self.weight, post_weight=self.post_weight, gate=self.gate, residual_scale=self.residual_scale, eps=self.eps)

    def extra_repr(self) -> str:
        return (f"{self.normalized_shape[0]}, eps={self.eps}, elementwise_affine={self.weight is not None}, post_norm={self.post_weight is not None}, "
                f"gate={self.gate is not None}, residual_scale={self.residual_scale}")
