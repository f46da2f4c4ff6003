"""The language-model example next to a twin in plain fp32 torch: same start, same batches, same schedule.

Tolerance: the twin differs by FP8 products, 16-bit activations and, with state_bits=8, moments of 3 bits of significand, none of
them biased; as for the other FP8 training runs here, the losses of the last steps may be 10 % apart."""
import os
import sys

import pytest
import torch
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu
STEPS, HIDDEN, LAYERS, VOCAB, TOKENS, LR = 80, 256, 2, 1000, 2048, 3e-3


def twin_losses(example):
    torch.manual_seed(0)
    model = example.LanguageModel(VOCAB, HIDDEN, LAYERS)
    own = {n: torch.nn.Parameter(p.as_subclass(torch.Tensor).detach().float().clone()) for n, p in model.named_parameters()}
    matrices = [p for n, p in own.items() if p.dim() == 2]
    rest = [p for p in own.values() if p.dim() == 1]
    opt = torch.optim.AdamW([dict(params=matrices, weight_decay=0.01), dict(params=rest, weight_decay=0.0)], lr=LR, betas=(0.9, 0.95))
    data = example.batches(VOCAB, 64, TOKENS // 64, "cuda", 1)
    losses = []
    for step in range(STEPS):
        for g in opt.param_groups:
            g["lr"] = LR * example.schedule(step, STEPS)
        tokens, labels = next(data)
        x = own["embedding.weight"][tokens]
        for i in range(LAYERS):
            y = F.layer_norm(x, (HIDDEN,), own[f"blocks.{i}.norm.weight"], own[f"blocks.{i}.norm.bias"])
            x = x + F.gelu(y @ own[f"blocks.{i}.up.weight"].t()) @ own[f"blocks.{i}.down.weight"].t()
        x = F.layer_norm(x, (HIDDEN,), own["norm.weight"], own["norm.bias"])
        loss = F.cross_entropy((x @ own["head"].t()).flatten(0, 1), labels.flatten())
        opt.zero_grad()
        loss.backward()
        torch.nn.utils.clip_grad_norm_(list(own.values()), 1.0)
        opt.step()
        losses.append(loss.item())
    return losses


def test_example_follows_plain_training():
    import train_language_model as example

    want = twin_losses(example)
    assert want[-1] < 0.5 * want[0]
    for bits in (32, 8):
        got = example.train(STEPS, HIDDEN, LAYERS, VOCAB, TOKENS, LR, bits)
        assert abs(got[0] - want[0]) < 0.02 * want[0]
        end, ref = sum(got[-10:]) / 10, sum(want[-10:]) / 10
        assert abs(end - ref) < 0.1 * ref, (bits, end, ref)
