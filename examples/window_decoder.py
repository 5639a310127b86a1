"""A decoder layer of window attention and a product-key memory: trained a few steps, then serving from a 4-bit cache.

    python examples/window_decoder.py [--steps 300] [--tokens 24]

The layer attends through a window with sinks (modelos_amd.window_attention),
reads a product-key memory (modelos_amd.pkm.memory.HashingMemory) in its
feed-forward slot, and learns sequences in which every token has one successor.
Then a left-padded batch of prompts goes through the same attention, its keys
and values into an Int4KVCache, and new tokens are decoded one at a time from
the cache. The script prints the losses and how many decoded tokens are right.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from modelos_amd.kv_cache import Int4KVCache  # noqa: E402
from modelos_amd.pkm.memory import HashingMemory  # noqa: E402
from modelos_amd.rmsnorm import QueryRMSNorm  # noqa: E402
from modelos_amd.window_attention import window_attention  # noqa: E402


class WindowAttention(nn.Module):
    """Grouped-query attention through a window with sinks; `cache` switches to decoding from 4 bits."""

    def __init__(self, width: int, heads: int, kv_heads: int, dim: int, window: int, sinks: int):
        super().__init__()
        self.heads, self.kv_heads, self.dim, self.window, self.sinks = heads, kv_heads, dim, window, sinks
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * dim, bias=False)
        self.out = nn.Linear(heads * dim, width, bias=False)

    def project(self, x):
        h = self.qkv(x).unflatten(-1, (-1, self.dim)).transpose(1, 2)  # [B, heads, T, dim], views of one tensor
        return h.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def merge(self, o):
        return self.out(o.transpose(1, 2).flatten(2))

    def forward(self, x, starts=None):
        q, k, v = self.project(x)
        return self.merge(window_attention(q, k, v, window=self.window, sinks=self.sinks, starts=starts)), k, v

    def decode(self, x, cache: Int4KVCache, table, lengths):
        """x [B, new, width]: the last tokens of sequences of `lengths` tokens, these among them."""
        q, k, v = self.project(x)
        new = x.shape[1]
        cache.append(k, v, table, lengths - new, torch.full_like(lengths, new))
        return self.merge(cache.attend(q, table, lengths, window=self.window, sinks=self.sinks))


class Decoder(nn.Module):
    def __init__(self, vocab=64, width=256, heads=4, kv_heads=2, dim=64, window=32, sinks=4, positions=512):
        super().__init__()
        self.embed, self.place = nn.Embedding(vocab, width), nn.Embedding(positions, width)
        self.norm1, self.norm2, self.norm3 = (QueryRMSNorm(width) for _ in range(3))
        self.attention = WindowAttention(width, heads, kv_heads, dim, window, sinks)
        self.memory = HashingMemory(input_dim=width, output_dim=width, mem_k_dim=128, mem_heads=2, mem_knn=8,
                                    mem_n_keys=64, mem_v_dim=64)
        self.memory.reset_parameters()
        nn.init.normal_(self.embed.weight, std=0.05)
        nn.init.normal_(self.place.weight, std=0.05)

    def inputs(self, tokens, positions):
        return self.embed(tokens) + self.place(positions)

    def head(self, x):
        x = x + self.memory(self.norm2(x))[0]
        return F.linear(self.norm3(x), self.embed.weight)

    def forward(self, tokens, positions, starts=None):
        x = self.inputs(tokens, positions)
        y, k, v = self.attention(self.norm1(x), starts)
        return self.head(x + y), k, v

    def decode(self, tokens, cache, table, lengths):
        x = self.inputs(tokens, (lengths - 1)[:, None].long())
        return self.head(x + self.attention.decode(self.norm1(x), cache, table, lengths))


def walks(batch: int, length: int, vocab: int, generator: torch.Generator) -> torch.Tensor:
    """Sequences in which every token has one successor: t -> (5 t + 7) mod vocab from a random first token."""
    rows = [torch.randint(0, vocab, (batch,), generator=generator)]
    for _ in range(length - 1):
        rows.append((5 * rows[-1] + 7) % vocab)
    return torch.stack(rows, 1)


def train(model: Decoder, steps: int, generator: torch.Generator, batch=16, length=129, vocab=64) -> list[float]:
    device = model.embed.weight.device
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3)
    positions = torch.arange(length - 1, device=device).expand(batch, -1)
    losses = []
    for _ in range(steps):
        tokens = walks(batch, length, vocab, generator).to(device)
        logits, _, _ = model(tokens[:, :-1], positions)
        loss = F.cross_entropy(logits.flatten(0, 1).float(), tokens[:, 1:].flatten())
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def generate(model: Decoder, prompts: torch.Tensor, starts: torch.Tensor, new: int, page: int = 16):
    """Greedy tokens [batch, new] behind left-padded prompts [batch, T]: the prompts at once, then one token at a time."""
    B, T = prompts.shape
    device = prompts.device
    counts = (T - starts).to(torch.int32)
    attention = model.attention
    width = -(-(T + new) // page)
    cache = Int4KVCache(B * width, attention.kv_heads, attention.dim, page_size=page,
                        dtype=attention.qkv.weight.dtype, device=device)
    table = torch.arange(B * width, dtype=torch.int32, device=device).view(B, width)
    positions = (torch.arange(T, device=device) - starts[:, None]).clamp_min(0)
    logits, k, v = model(prompts, positions, starts)
    # the prompts' own tokens to the front, as the cache counts from each sequence's first
    front = (torch.arange(T, device=device) + starts[:, None]).clamp_max(T - 1)[:, None, :, None]
    k, v = (x.gather(2, front.expand(-1, x.shape[1], -1, x.shape[3])) for x in (k, v))
    cache.append(k, v, table, torch.zeros_like(counts), counts)
    token, lengths, out = logits[:, -1:].argmax(-1), counts, []
    for _ in range(new):
        out.append(token)
        lengths = lengths + 1
        token = model.decode(token, cache, table, lengths)[:, -1:].argmax(-1)
    return torch.cat(out, 1)


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--tokens", type=int, default=24)
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    generator = torch.Generator().manual_seed(0)
    model = Decoder().to("cuda", torch.bfloat16)
    losses = train(model, args.steps, generator)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} after {len(losses)} steps")
    T, B = 100, 8
    text = walks(B, T + args.tokens, 64, generator).to("cuda")
    starts = torch.arange(B, dtype=torch.int32, device="cuda") * 5  # left padding of 0 to 35 tokens
    out = generate(model, text[:, :T], starts, args.tokens)
    right = (out == text[:, T:]).float().mean().item()
    print(f"decoded {args.tokens} tokens of {B} sequences from the 4-bit cache, {100 * right:.0f} % as the sequences go on")
    return {"losses": losses, "right": right}


if __name__ == "__main__":
    main()
