"""Trains a small language model on one GPU: FP8 linears in its blocks, and beside them the package's layer norm, its
vocabulary projection with cross entropy, and its AdamW, with moments in 8 bits unless --state-bits 32.

    python examples/train_language_model.py [--steps 200] [--hidden 512] [--layers 4] [--vocab 8000] [--tokens 4096] [--heads 8 --kv-heads 2]

The text is synthetic: every token is followed by one of four others, chosen at random from a fixed table, so that a model that has
learned the table reaches a loss of log(4) = 1.386.  The first quarter of every sequence counts as prompt (label -100).

How the parts fit.  The blocks' FP8Linears keep bf16 masters and re-quantise them after every optimizer step
(`attach_requantize_hook`).  The head is not FP8: its weight is an fp32 master whose bf16 copy, which the projection reads, is
written by the optimizer in the same pass (`copies`).  The clipping factor stays on the device (`grad_scale`).

With --heads the blocks are those of a decoder: attention with grouped heads and rotary positions over the packed sequences of the
batch, and one fused pass for the residual and the norm between an attention, an MLP and the next attention.
"""
import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from nanotron_amd.fp8 import FP8Linear  # noqa: E402
from nanotron_amd.fp8.optim import attach_requantize_hook, requantize_fp8_weights  # noqa: E402
from nanotron_amd.nn import LayerNorm, RMSNorm, RotaryEmbedding, attention, linear_cross_entropy  # noqa: E402
from nanotron_amd.optim import AdamW  # noqa: E402

BRANCHES = 4


class Block(nn.Module):
    """A norm and an MLP on the residual stream.  (No attention: in this language the next token depends on the last alone.)"""

    def __init__(self, hidden: int, device):
        super().__init__()
        self.norm = LayerNorm(hidden, device=device)
        fp8 = dict(bias=False, device=device, dtype=torch.bfloat16, out_dtype=torch.bfloat16, delayed_scaling=True)
        self.up, self.down = FP8Linear(hidden, 4 * hidden, **fp8), FP8Linear(4 * hidden, hidden, **fp8)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = self.norm(x)
        return x + self.down(nn.functional.gelu(self.up(y)))


class DecoderBlock(nn.Module):
    """Attention and an MLP on the residual stream.  What a block hands on is the MLP's output and the stream it belongs to, which the
    norm of the next one adds up."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, device):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, hidden // heads
        self.norm, self.mlp_norm = RMSNorm(hidden, device=device), RMSNorm(hidden, device=device)
        self.rotary = RotaryEmbedding(self.dim, device=device)
        fp8 = dict(bias=False, device=device, dtype=torch.bfloat16, out_dtype=torch.bfloat16, delayed_scaling=True)
        self.qkv, self.out = FP8Linear(hidden, (heads + 2 * kv_heads) * self.dim, **fp8), FP8Linear(hidden, hidden, **fp8)
        self.up, self.down = FP8Linear(hidden, 4 * hidden, **fp8), FP8Linear(4 * hidden, hidden, **fp8)

    def forward(self, x, residual, positions, cu_seqlens):
        # (in front of the first block there is no residual yet: the stream is x itself)
        y, residual = (self.norm(x), x) if residual is None else self.norm(x, residual)
        q, k, v = self.qkv(y).unflatten(-1, (-1, self.dim)).split([self.heads, self.kv_heads, self.kv_heads], 1)
        q, k = self.rotary(q, k, positions)
        y, residual = self.mlp_norm(self.out(attention(q, k, v, cu_seqlens=cu_seqlens).flatten(1)), residual)
        return self.down(nn.functional.gelu(self.up(y))), residual


class LanguageModel(nn.Module):
    def __init__(self, vocab: int, hidden: int, layers: int, device="cuda", heads: int = 0, kv_heads: int = 0):
        super().__init__()
        self.decoder = heads > 0
        self.embedding = nn.Embedding(vocab, hidden, device=device, dtype=torch.bfloat16)
        self.blocks = nn.ModuleList(DecoderBlock(hidden, heads, kv_heads or heads, device) if heads else Block(hidden, device) for _ in range(layers))
        self.norm = RMSNorm(hidden, device=device) if heads else LayerNorm(hidden, device=device)
        # the projection as the loss reads it; its fp32 master belongs to the optimizer
        self.head = nn.Parameter(torch.randn(vocab, hidden, device=device).mul_(hidden ** -0.5).bfloat16())
        for lin in self.blocks.modules():
            if isinstance(lin, FP8Linear):
                with torch.no_grad():
                    lin.weight.as_subclass(torch.Tensor).normal_(std=lin.in_features ** -0.5)
        requantize_fp8_weights(self)

    def forward(self, tokens: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        if not self.decoder:
            x = self.embedding(tokens)
            for b in self.blocks:
                x = b(x)
            return linear_cross_entropy(self.norm(x), self.head, labels)
        # the batch's sequences end to end, each counted from 0
        count, length = tokens.shape
        positions = torch.arange(length, device=tokens.device).repeat(count)
        cu_seqlens = torch.arange(count + 1, device=tokens.device, dtype=torch.int32) * length
        x, residual = self.embedding(tokens.flatten()), None
        for b in self.blocks:
            x, residual = b(x, residual, positions, cu_seqlens)
        y = self.norm(x) if residual is None else self.norm(x, residual)[0]
        return linear_cross_entropy(y, self.head, labels.flatten())


def optimizer_of(model: LanguageModel, lr: float, state_bits: int) -> AdamW:
    """AdamW over everything: the head through its fp32 master, matrices with weight decay, the rest without."""
    master = nn.Parameter(model.head.detach().float())
    matrices = [p for n, p in model.named_parameters() if p.dim() == 2 and n != "head"]
    rest = [p for p in model.parameters() if p.dim() == 1]
    opt = AdamW([dict(params=matrices, weight_decay=0.01), dict(params=rest, weight_decay=0.0),
                 dict(params=[master], copies=[model.head], weight_decay=0.01)], lr=lr, betas=(0.9, 0.95), state_bits=state_bits)
    attach_requantize_hook(opt, model)
    return opt


def batches(vocab: int, length: int, count: int, device, seed: int):
    """Endless batches of (tokens, labels) from the table."""
    g = torch.Generator(device=device).manual_seed(seed)
    table = torch.randint(0, vocab, (vocab, BRANCHES), generator=g, device=device)
    while True:
        t = torch.empty(count, length + 1, dtype=torch.int64, device=device)
        t[:, 0] = torch.randint(0, vocab, (count,), generator=g, device=device)
        pick = torch.randint(0, BRANCHES, (count, length), generator=g, device=device)
        for i in range(length):
            t[:, i + 1] = table[t[:, i], pick[:, i]]
        labels = t[:, 1:].clone()
        labels[:, :length // 4] = -100
        yield t[:, :-1], labels


def clipping_factor(grads, limit: float) -> torch.Tensor:
    """min(1, limit / norm) as one value on the device."""
    norm = torch.stack([g.float().norm() for g in grads]).norm()
    return (limit / (norm + 1e-6)).clamp_max_(1.0).reshape(1)


def schedule(step: int, steps: int) -> float:
    """Share of the learning rate: 20 steps up, then along a cosine to nothing."""
    return min(1.0, (step + 1) / 20) * 0.5 * (1 + math.cos(math.pi * step / steps))


def train(steps: int = 200, hidden: int = 512, layers: int = 4, vocab: int = 8000, tokens: int = 4096, lr: float = 3e-3, state_bits: int = 8, clip: float = 1.0,
          seed: int = 0, report=None, heads: int = 0, kv_heads: int = 0):
    """Returns the losses of the steps, as floats."""
    torch.manual_seed(seed)
    model = LanguageModel(vocab, hidden, layers, heads=heads, kv_heads=kv_heads)
    opt = optimizer_of(model, lr, state_bits)
    length = min(64, tokens)
    data = batches(vocab, length, tokens // length, "cuda", seed + 1)
    losses = []
    for step in range(steps):
        for group in opt.param_groups:
            group["lr"] = lr * schedule(step, steps)
        loss = model(*next(data))
        loss.backward()
        grads = [opt.grad_of(p, copy).as_subclass(torch.Tensor) for p, copy in opt.params_and_copies()]
        opt.step(grad_scale=clipping_factor(grads, clip))
        opt.zero_grad()
        losses.append(loss.detach())
        if report and (step % 20 == 19 or step == 0):
            report(f"step {step + 1:4d}  loss {loss.item():.4f}")
    return [x.item() for x in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("steps", 200), ("hidden", 512), ("layers", 4), ("vocab", 8000), ("tokens", 4096), ("state-bits", 8), ("seed", 0), ("heads", 0), ("kv-heads", 0)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--lr", type=float, default=3e-3)
    a = ap.parse_args()
    train(a.steps, a.hidden, a.layers, a.vocab, a.tokens, a.lr, a.state_bits, seed=a.seed, report=lambda line: print(line, flush=True), heads=a.heads,
          kv_heads=a.kv_heads)


if __name__ == "__main__":
    main()
