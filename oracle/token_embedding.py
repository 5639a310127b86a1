"""Token embedding and its table's gradient in 64 bits on the CPU, and how far kernels may lie from them."""
from __future__ import annotations

import torch


def embedding(ids, w, scale: float):
    """scale * w[ids]; ids outside the table read zeros."""
    there = (ids >= 0) & (ids < w.shape[0])
    out = w.double()[torch.where(there, ids, 0).long()] * scale if w.shape[0] else torch.zeros((*ids.shape, w.shape[1])).double()
    return torch.where(there[..., None], out, 0.0)


def gradient(ids, grad, rows: int, scale: float, padding: int | None):
    """(dW, the same sums over the terms' sizes, tokens of each row)."""
    ids, grad = ids.flatten().long(), grad.double().flatten(0, -2)
    kept = (ids >= 0) & (ids < rows) & (ids != (-1 if padding is None else padding))
    dw = torch.zeros((rows, grad.shape[1]), dtype=torch.float64)
    size = dw.clone()
    dw.index_add_(0, ids[kept], grad[kept])
    size.index_add_(0, ids[kept], grad[kept].abs())
    return dw * scale, size * abs(scale), torch.bincount(ids[kept], minlength=rows)


def allowed(value, size, terms, dtype):
    """A result rounded once to dtype, of `terms` float32 additions of numbers that sum to `size` in absolute value (and
    a float32 product)."""
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    sums = (terms + 2) * 2.0**-24 * size
    return u * (value.abs() + sums) + sums + tiny
