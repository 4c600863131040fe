"""Learns an encoder whose embeddings align: the whole path from tokens to a soft
Smith-Waterman value and back.

Pairs of token sequences, one a mutated copy of the other or not, go through a small
encoder (d2p_amd.SequenceAttention: norm and rotation of queries and keys, attention with a
learned relative position bias and dropout); the products of their embeddings are the score
matrix of d2p_amd.soft_sw, and the encoder learns to give related pairs the higher values.
Then a causal layer reads a sequence token by token from its cache, and gives what it gives
for the sequence as a whole.

    python examples/train_encoder.py [--steps 60] [--length 96] [--batch 32]
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import d2p_amd  # noqa: E402

TOKENS = 21     # twenty letters and padding


class Encoder(nn.Module):
    def __init__(self, dim=128, heads=4, layers=2):
        super().__init__()
        self.embed = nn.Embedding(TOKENS, dim)
        self.layers = nn.ModuleList(
            d2p_amd.SequenceAttention(dim, heads, num_buckets=32, max_distance=64, dropout=0.1)
            for _ in range(layers))
        self.norms = nn.ModuleList(nn.LayerNorm(dim) for _ in range(layers))
        self.out = nn.Linear(dim, 32)

    def forward(self, tokens, lengths):
        x = self.embed(tokens)
        for norm, layer in zip(self.norms, self.layers):
            x = x + layer(norm(x), lengths)
        return self.out(x)


def pairs(batch, length, device, generator):
    """tokens a, b [batch, length], lengths [batch, 2], related [batch]: every other b is a
    with a fifth of its letters changed and a stretch of them left out."""
    def letters(*shape):
        return torch.randint(0, TOKENS - 1, shape, generator=generator)
    a, b = letters(batch, length), letters(batch, length)
    lengths = torch.randint(length // 2, length + 1, (batch, 2), generator=generator)
    for n in range(0, batch, 2):
        cut = int(torch.randint(0, length // 4, (1,), generator=generator))
        copy = torch.cat((a[n, :cut], a[n, cut + 3:]))
        change = torch.rand(copy.shape, generator=generator) < 0.2
        b[n, :len(copy)] = torch.where(change, letters(len(copy)), copy)
    for tokens, long in ((a, lengths[:, 0]), (b, lengths[:, 1])):
        tokens[torch.arange(length)[None] >= long[:, None]] = TOKENS - 1
    related = (torch.arange(batch) % 2 == 0).float()
    return a.to(device), b.to(device), lengths.to(torch.int32).to(device), related.to(device)


def train(steps=60, batch=32, length=96, device="cuda", seed=0, autocast=True, report=print):
    torch.manual_seed(seed)
    generator = torch.Generator().manual_seed(seed)
    model = Encoder().to(device)
    scale = nn.Parameter(torch.tensor([0.05, -2.0], device=device))   # of the value, and its zero
    optimizer = torch.optim.AdamW([*model.parameters(), scale], lr=2e-3)
    losses = []
    for step in range(steps):
        a, b, lengths, related = pairs(batch, length, device, generator)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            x, y = model(a, lengths[:, 0]), model(b, lengths[:, 1])
        scores = F.normalize(x.float(), dim=-1) @ F.normalize(y.float(), dim=-1).transpose(1, 2)
        value = d2p_amd.soft_sw(4.0 * scores - 1.0, gap=-1.0, temperature=1.0,
                                lengths=lengths).value
        loss = F.binary_cross_entropy_with_logits(scale[0] * value + scale[1], related)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            report(f"step {step:4d}  loss {losses[-1]:.4f}")
    return losses


@torch.no_grad()
def stream(tokens=24, batch=2, dim=128, device="cuda", seed=0, report=print):
    """The largest difference between a causal layer's outputs for a whole sequence and for
    the same sequence token by token."""
    torch.manual_seed(seed)
    layer = d2p_amd.SequenceAttention(dim, 8, kv_heads=2, causal=True, num_buckets=16,
                                      max_distance=32).to(device).eval()
    nn.init.normal_(layer.bias)
    x = torch.randn(batch, tokens, dim, device=device)
    whole = layer(x)
    cache = layer.new_cache(batch, tokens)
    steps = torch.cat([layer.step(x[:, n:n + 1], cache) for n in range(tokens)], 1)
    worst = float((whole - steps).abs().max())
    report(f"whole sequence against {tokens} single tokens: largest difference {worst:.2e}")
    return worst


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--length", type=int, default=96)
    parser.add_argument("--batch", type=int, default=32)
    args = parser.parse_args()
    train(args.steps, args.batch, args.length)
    stream()
