from typing import Optional

import torch
from torch import nn

from nanotron_amd import _ops


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits `x @ weight.T` against `labels`, with the logits never in memory.

    x [..., hidden] and weight [vocab, hidden]: both bfloat16 or both float16; labels [...]: int64.  The products run on
    the matrix cores with fp32 sums; maxima, sums and losses are fp32.  Labels equal to `ignore_index` have loss 0 and no
    gradient and are left out of the mean, which is 0 if all are ignored.  Any other label outside [0, vocab) makes its
    token's loss, and with it the result and the gradients it reaches, NaN: nothing is read back to raise an error.

    reduction "mean" or "sum": a float32 scalar.  Both gradients are made in the forward call, where the softmax is at
    hand (three products in all, no recomputation), and handed to autograd once: a second backward through the same loss
    raises RuntimeError.  bfloat16 gradients are rounded there, and a second time by a factor from above that is no power of
    two (a loss divided by three accumulated batches); float16 ones are fp32 until then.  "none": the float32 losses of the
    tokens, without gradients (ValueError if any are wanted).

    Memory beside the gradients, freed when the call returns: 2 bytes a logit for at most 2 GiB worth of tokens at a time, sums
    of the gradient of x in fp32 (4 bytes an element, at most 2 GiB at a time, or 256 MiB where there are few tokens), a copy of
    x, and one of weight if its rows do not begin on 16-byte boundaries or lie more than 2^22 elements apart.
    Tokens beyond 2 GiB of logits go in pieces, with the gradient of the weight summed in fp32 (4 bytes an element, freed likewise),
    which float16 inputs always use, so that a loss scale cannot overflow or underflow them."""
    return _ops.host.linear_cross_entropy(x, weight, labels, ignore_index, reduction)


class LinearCrossEntropy(nn.Module):
    """A vocabulary projection and its loss: `weight` [vocab_size, hidden_size] as nn.Linear keeps it, forward(x, labels)
    = `linear_cross_entropy`."""

    def __init__(self, hidden_size: int, vocab_size: int, ignore_index: int = -100, reduction: str = "mean",
                 device: Optional[torch.device] = None, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.ignore_index, self.reduction = ignore_index, reduction
        self.weight = nn.Parameter(torch.empty(vocab_size, hidden_size, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=0.02)

    def forward(self, x: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(x, self.weight, labels, ignore_index=self.ignore_index, reduction=self.reduction)

    def extra_repr(self) -> str:
        return f"hidden_size={self.weight.shape[1]}, vocab_size={self.weight.shape[0]}, ignore_index={self.ignore_index}, reduction={self.reduction!r}"
