from typing import Optional

import torch
from torch import nn

from nanotron_amd import _ops


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer normalisation over the last dimension: `(x - mean) / sqrt(var + eps) * weight + bias`.

    x: float32, float16 or bfloat16, any number of dimensions; the result has its type.  weight and bias ([x.shape[-1]],
    each optional) are float32 or of the type of x.  Arithmetic is fp32; the gradients of weight and bias are
    summed in fp32 within a workgroup and in 64 bits over them, in an order that depends on the sizes alone, so gradients
    repeat bit for bit.  Rows that are dense in themselves (a slice of a wider 2-D tensor) are read where they are.  Up to 32768 columns of
    a 16-bit x, 16384 of float32.  ValueError / TypeError for what does not fit; differentiable once."""
    return _ops.host.layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """`layer_norm` as a module, with the constructor of torch.nn.LayerNorm for one normalised dimension.  `dtype` is that
    of weight and bias, which may stay float32 beside 16-bit activations."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device: Optional[torch.device] = None, dtype: Optional[torch.dtype] = None):
        super().__init__()
        if not isinstance(normalized_shape, int):
            if len(normalized_shape) != 1:
                raise ValueError(f"LayerNorm normalises the last dimension, got normalized_shape={normalized_shape}")
            normalized_shape = normalized_shape[0]
        self.normalized_shape, self.eps = (normalized_shape,), eps
        made = dict(device=device, dtype=dtype)
        self.weight = nn.Parameter(torch.ones(normalized_shape, **made)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(normalized_shape, **made)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"the last dimension of x must be {self.normalized_shape[0]}, got shape {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.normalized_shape[0]}, eps={self.eps}, elementwise_affine={self.weight is not None}"
