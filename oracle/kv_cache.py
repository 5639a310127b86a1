"""The 4-bit key / value cache on the CPU: quantised vectors, their codes' places, numbers read back."""
from __future__ import annotations

import torch

GROUP = 32


def quantise(x: torch.Tensor):
    """codes (int64) like x, steps and minima [..., dim / 32] of x's type."""
    g = x.double().unflatten(-1, (-1, GROUP))
    m, top = g.amin(-1), g.amax(-1)
    s = ((top - m) / 15).to(x.dtype)
    step = s.double()[..., None]
    c = torch.where(step > 0, torch.round((g - m[..., None]) / torch.where(step > 0, step, 1.0)), 0.0)
    return c.clamp(0, 15).long().flatten(-2), s, m.to(x.dtype)


def values(c: torch.Tensor, s: torch.Tensor, m: torch.Tensor) -> torch.Tensor:
    """The numbers in 64 bits."""
    c = c.double().unflatten(-1, (-1, GROUP))
    return (m.double()[..., None] + s.double()[..., None] * c).flatten(-2)


def pack(c: torch.Tensor) -> torch.Tensor:
    """Bytes [..., dim / 2] of codes [..., dim], one nibble at a time."""
    D = c.shape[-1]
    out = torch.zeros((*c.shape[:-1], D // 2), dtype=torch.int64)
    for d in range(D):
        w, i = d % 16, d // 16
        bit = 32 * w + 4 * (i // 2 + 4 * (i % 2)) if D == 128 else 16 * w + 4 * i
        out[..., bit // 8] |= c[..., d] << (bit % 8)
    return out.to(torch.uint8)


def unpack(b: torch.Tensor, D: int) -> torch.Tensor:
    cols = []
    for d in range(D):
        w, i = d % 16, d // 16
        bit = 32 * w + 4 * (i // 2 + 4 * (i % 2)) if D == 128 else 16 * w + 4 * i
        cols.append((b[..., bit // 8].long() >> (bit % 8)) & 15)
    return torch.stack(cols, -1)


def sequence(codes: torch.Tensor, params: torch.Tensor, pages: list, n: int, side: int) -> torch.Tensor:
    """[heads, n, dim] in 64 bits: positions 0 .. n - 1 of a sequence whose table row is `pages`."""
    P, D = codes.shape[3], 2 * codes.shape[4]
    out = torch.zeros((codes.shape[2], n, D), dtype=torch.float64)
    for i in range(0, n, P):
        p, e = int(pages[i // P]) if i // P < len(pages) else -1, min(n - i, P)
        if 0 <= p < codes.shape[1]:
            s, m = (x.transpose(-1, -2)[:, :e] for x in params[side, p].unbind(1))
            out[:, i : i + e] = values(unpack(codes[side, p, :, :e], D), s, m)
    return out
