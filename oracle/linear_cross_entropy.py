"""Cross entropy of a linear layer in 64 bits on the CPU, its gradients from the formulas, and how far 16-bit kernels may lie
from them."""
from __future__ import annotations

import torch


def loss_and_gradients(x, w, labels, ignore: int, reduction: str, grad=None, each: bool = False):
    """x [n, D], w [V, D], labels [n]: values (loss, dx, dW) and bounds of the same shapes.

    The bounds are those of a kernel that sums in float32, rounds the logits' gradients once to x's type (relative error u)
    for the products with w and x, and rounds its results once. grad: float64 [] or [n]. each: f16's logits' gradients are
    held in units of their own token's gradient, not of the largest.
    """
    n, D = x.shape
    V = w.shape[0]
    u = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * u
    f = 2.0**-24
    live = (labels != ignore) & (labels >= 0) & (labels < V)
    x = torch.where(live[:, None], x.double(), 0.0)
    w = w.double()
    y = torch.where(live, labels, 0).long()
    logits = x @ w.T
    lse = torch.logsumexp(logits, 1)
    losses = torch.where(live, lse - logits.gather(1, y[:, None]).squeeze(1), 0.0)
    # float32 logits: D products and sums; log2 e, the exponent's and the exponential's rounding; the sum of V exponentials
    size = x.abs() @ w.abs().T
    e_logit = f * ((D + 2) * size + 4 * logits.abs() + 4)
    e_lse = (e_logit.max(1).values + f * (4 * lse.abs() + 2 * V**0.5 + 16))
    e_loss = torch.where(live, e_lse + e_logit.gather(1, y[:, None]).squeeze(1) + 4 * f * losses.abs(), 0.0)
    count = max(1, int(live.sum()))
    scale = 1 / count if reduction == "mean" else 1.0
    value = losses if reduction == "none" else losses.sum() * scale
    bound = e_loss if reduction == "none" else (e_loss.sum() + f * 40 * losses.sum()) * scale
    if grad is None:
        return value, bound
    g = torch.where(live, (grad * scale).expand(n), 0.0)[:, None]
    p = (logits - lse[:, None]).exp()
    onehot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    d = (p - onehot) * g
    # d: the exponential's error, one float32 rounding more for the label's, the rounding to 16 bits, what f16 cannot hold
    # (2^-24 2^-14 of the largest gradient)
    unit = g.abs() if each else g.abs().max()
    e_d = g.abs() * (p * (e_logit + e_lse[:, None]) + f * 4 * (p + onehot)) + u * d.abs() + f * 2.0**-13 * unit
    dx, dw = d @ w, d.T @ x
    e_dx = e_d @ w.abs() + f * 64 * (d.abs() @ w.abs())
    e_dw = e_d.T @ x.abs() + f * 64 * (d.abs().T @ x.abs())
    if each:  # the powers of two between the tokens' go to x: the largest product with its gradient (within a factor of 4) is
        # 2^15, f16's rounding 2^-25
        e_dw = e_dw + 2.0**-38 * (g.abs() * x.abs()).max() * (p - onehot).abs().T @ live[:, None].double().expand_as(x)
    # float32 sums of n or V numbers: 64 roundings stand for the blocks of a matrix product and its splits, whose
    # errors add like a random walk
    return ((value, dx, dw),
            (bound, e_dx + u * (dx.abs() + e_dx) + tiny, e_dw + u * (dw.abs() + e_dw) + tiny))
