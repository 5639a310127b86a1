"""An AdamW step on the CPU: in 64 bits, and the rounded states that a kernel has to hold bit for bit."""
from __future__ import annotations

import torch

BLOCK = 256
TOP = 448.0


def step(p, g, m, v, t: int, lr, betas, eps, decay):
    """(p, m, v) after step number t, in 64 bits."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    root = (v / (1 - betas[1] ** t)).sqrt()
    return p * (1 - lr * decay) - lr / (1 - betas[0] ** t) * m / (root + eps), m, v


def moments(g, m, v, betas):
    """m and v in float32, rounded as the kernels round: b m first, then one operation with the gradient's part."""
    fused = lambda a, x, y: (torch.tensor(a, dtype=torch.float32).double() * x.double() + y.double()).float()
    b = [torch.tensor(x, dtype=torch.float32) for x in betas]
    return fused(1 - betas[0], g, b[0] * m), fused(1 - betas[1], g * g, b[1] * v)


def _blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)


def dither(n: int, t: int):
    """(of m, of r), [n]."""
    x = (torch.arange(n) * 2654435761 + t * 2246822519) % (1 << 32)
    return (x >> 12) * 2.0**-20, (x % (1 << 20)) * 2.0**-20


def hold(x, u, least: float):
    """(codes as the numbers they are, steps) of float32 x: a = |x| / step, floor(a 2^(3 - e) + u) 2^(e - 3)."""
    top = _blocks(x.abs()).amax(1)
    flat = top < 2.0**-110
    step = torch.where(flat, 0.0, top * torch.tensor(1 / TOP, dtype=torch.float32))
    a = _blocks(x.abs()).double() / torch.where(flat, 1.0, step).double()[:, None]
    a = torch.where(flat[:, None], 0.0, a)
    e = (torch.frexp(a).exponent - 1).clamp_min(-6)
    held = torch.ldexp(torch.floor(torch.ldexp(a, 3 - e) + _blocks(u)), e - 3).clamp_max(TOP)
    held = torch.where(flat[:, None], 0.0, held)
    if least:
        held = torch.where(a > 0, held.clamp_min(least), 0.0)
    held = torch.where(_blocks(x) < 0, -held, held)
    return held.reshape(-1)[: x.numel()].view(x.shape).float(), step


def numbers(codes, steps):
    """float32 numbers of e4m3 codes and their blocks' steps."""
    return (_blocks(codes.float()) * steps[:, None]).reshape(-1)[: codes.numel()].view(codes.shape)
