import math
from typing import Mapping, Optional, Tuple

import torch
from torch import nn

from nanotron_amd import _ops


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *, interleaved: bool = False,
           scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions: turns pair i of the first `2 * len(frequencies)` elements of every head of q and k by
    `angle = position * frequencies[i]`, `(a, b) -> (a cos - b sin, b cos + a sin) * scale`, and copies the elements behind them.

    q [..., heads, head_dim] and k [..., kv_heads, head_dim] (or None): float32, float16 or bfloat16, of one type; views of a wider tensor, as
    the parts of one linear's output, are read where they are.  positions: int64 or int32, of the shape of q in front of its heads, or
    of the last of these dimensions, which the others share; any values, there is no table that bounds them.  frequencies: float64 [pairs],
    radians a position.  The elements of a pair are `len(frequencies)` apart, or neighbours if `interleaved`.  Angles are made in 64
    bits, sines, cosines and products in fp32, rounded once.  Returns (q, k) rotated, dense.  Gradients reach q and k, by the
    rotation the other way; ValueError / TypeError for what does not fit; differentiable once."""
    out = _ops.host.rotary(q, k, positions, frequencies, interleaved, scale)
    return out[0], (out[1] if k is not None else None)


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[Mapping] = None, device: Optional[torch.device] = None) -> Tuple[torch.Tensor, float]:
    """(frequencies, scale) for `rotary`: float64 `base ** (-2 i / dim)` for the dim / 2 pairs of `dim` elements, and the factor of sines and
    cosines, for a model made for contexts of `original` positions and used for `factor` times as many.  `scaling`: None, or a
    dict with "kind" and what that kind needs:

    "linear"      (factor): every position counts 1 / factor.
    "base"        (factor): the base grows by factor ** (dim / (dim - 2)), so that the slowest pair turns 1 / factor as fast and the fastest as before.
    "wavelength"  (factor, original, low=1.0, high=4.0): pairs whose wavelength is above original / low positions are slowed by factor,
                  those below original / high stay, and between them the two are blended linearly in original / wavelength.
    "yarn"        (factor, original, slow=1.0, fast=32.0, scale=0.1 * log(factor) + 1): pairs that turn less than `slow` times over
                  `original` positions are slowed by factor, those that turn more than `fast` times stay, with a linear ramp over the
                  pairs between; sines and cosines are multiplied by scale."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and positive, got {dim}")
    if not base > 1:
        raise ValueError(f"base must be above 1, got {base}")
    given = dict(scaling or {})
    kind = given.pop("kind", None)
    allowed = {None: (), "linear": ("factor",), "base": ("factor",), "wavelength": ("factor", "original", "low", "high"),
               "yarn": ("factor", "original", "slow", "fast", "scale")}
    if kind not in allowed:
        raise ValueError(f"scaling['kind'] must be one of {[k for k in allowed if k]}, got {kind!r}")
    if set(given) - set(allowed[kind]):
        raise ValueError(f"scaling of kind {kind!r} takes {list(allowed[kind])}, got {sorted(given)}")
    missing = [k for k in ("factor", "original") if k in allowed[kind] and k not in given]
    if missing:
        raise ValueError(f"scaling of kind {kind!r} needs {missing}")
    for k, v in given.items():
        if not (isinstance(v, (int, float)) and v > 0 and math.isfinite(v)):
            raise ValueError(f"scaling[{k!r}] must be a positive number, got {v!r}")
    factor, scale = float(given.get("factor", 1.0)), 1.0
    if kind == "base":
        base *= factor ** (dim / (dim - 2)) if dim > 2 else 1.0
    f = torch.arange(0, dim, 2, dtype=torch.float64).div_(-dim)
    f = torch.pow(torch.tensor(base, dtype=torch.float64), f)
    if kind == "linear":
        f /= factor
    elif kind == "wavelength":
        low, high = given.get("low", 1.0), given.get("high", 4.0)
        if not high > low:
            raise ValueError(f"scaling['high'] must be above scaling['low'], got {high} and {low}")
        stay = ((given["original"] * f / (2 * math.pi) - low) / (high - low)).clamp_(0, 1)
        f = f * stay + f / factor * (1 - stay)
    elif kind == "yarn":
        slow, fast = given.get("slow", 1.0), given.get("fast", 32.0)
        if not fast > slow:
            raise ValueError(f"scaling['fast'] must be above scaling['slow'], got {fast} and {slow}")

        def pair(turns):   # the pair that turns so often over the original positions
            return dim * math.log(given["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(0, math.floor(pair(fast))), min(dim - 1, math.ceil(pair(slow)))
        slowed = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp_(0, 1)
        f = f / factor * slowed + f * (1 - slowed)
        scale = float(given.get("scale", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    return f.to(device) if device is not None else f, scale


class RotaryEmbedding(nn.Module):
    """`rotary` with its frequencies: forward(q, k, positions) -> (q, k).  `rotary_dim` elements of each head turn (all by default);
    base and scaling as in `rotary_frequencies`."""

    def __init__(self, head_dim: int, base: float = 10000.0, scaling: Optional[Mapping] = None, *, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 device: Optional[torch.device] = None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim > head_dim:
            raise ValueError(f"rotary_dim must be at most head_dim {head_dim}, got {rotary_dim}")
        self.head_dim, self.rotary_dim, self.interleaved, self.base = head_dim, rotary_dim, interleaved, base
        frequencies, self.scale = rotary_frequencies(rotary_dim, base, scaling, device)
        self.register_buffer("frequencies", frequencies, persistent=False)

    def _apply(self, fn, recurse=True):
        # a model that is cast to 16 bits keeps its frequencies in 64: only their device follows
        kept = self.frequencies
        super()._apply(fn, recurse)
        if self.frequencies.dtype != torch.float64:
            self.frequencies = kept.to(self.frequencies.device)
        return self

    def forward(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"heads must have {self.head_dim} elements, got shape {tuple(q.shape)}")
        return rotary(q, k, positions, self.frequencies, interleaved=self.interleaved, scale=self.scale)

    def extra_repr(self) -> str:
        return f"{self.head_dim}, base={self.base}, rotary_dim={self.rotary_dim}, interleaved={self.interleaved}, scale={self.scale}"
