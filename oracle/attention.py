"""Attention through a window with sinks in 64 bits on the CPU, its gradients from the formulas, and how far 16-bit
kernels may lie from them."""
from __future__ import annotations

import torch


def visible(T: int, start: int, end: int, window: int | None, sinks: int) -> torch.Tensor:
    """[T, T] truth values: may query p (row) see key j."""
    p, j = torch.arange(T)[:, None], torch.arange(T)[None]
    near = p - j < (window if window is not None else T + 1)
    return (j >= start) & (j <= p) & (p < end) & (near | (j - start < sinks))


def masks(B: int, T: int, window, sinks, starts=None, ends=None) -> torch.Tensor:
    """[B, 1, T, T], bounds clamped to the tokens as the kernels do."""
    clamp = lambda x: min(max(int(x), 0), T)
    return torch.stack([visible(T, 0 if starts is None else clamp(starts[b]), T if ends is None else clamp(ends[b]),
                                window, sinks) for b in range(B)])[:, None]


def attention(q, k, v, mask, scale=None, grad=None):
    """q [B, H, Q, D], k, v [B, Hk, N, D], mask [B, 1, Q, N]: out, and with grad (dq, dk, dv) too.

    Returns (values, bounds): bounds[i] is how far a kernel may lie from values[i] that rounds softmax weights and
    their gradients to q's type once (relative error u), sums in 32 bits and rounds its results once. dS takes the
    rounded output's error through delta."""
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * u  # half the step of its subnormal numbers
    B, H, Q, D = q.shape
    G = H // k.shape[1]
    scale = D**-0.5 if scale is None else scale
    q, kk, vv = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    # what no query sees takes no part, whatever it holds
    seen = mask.any(-2)[..., None]
    live = mask.any(-1)[..., None]
    q, kk, vv = torch.where(live, q, 0.0), torch.where(seen, kk, 0.0), torch.where(seen, vv, 0.0)
    s = q @ kk.transpose(-1, -2) * scale
    # float32 sums and exponentials: D products and the logit's own size, in units of 2^-24
    es = 2.0**-24 * ((D + 8) * scale * (q.abs() @ kk.abs().transpose(-1, -2)) + 4 * s.abs() + 8)
    s = torch.where(mask, s, -torch.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-1e300)
    e = torch.where(mask, torch.exp(s - top), 0.0)
    P = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    ep = P * (2 * torch.where(mask, es, 0.0).amax(-1, keepdim=True) + 2.0**-20)  # of P, before its rounding
    out = P @ vv
    rounded = u * P + ep + torch.where(mask, tiny, 0.0)
    eo = rounded @ vv.abs() + u * out.abs() + tiny
    if grad is None:
        return [out], [eo]
    g = torch.where(live, grad.double(), 0.0)
    dP = g @ vv.transpose(-1, -2)
    edp = 2.0**-24 * D * (g.abs() @ vv.abs().transpose(-1, -2))
    delta = (g * out).sum(-1, keepdim=True)
    edelta = (g.abs() * eo).sum(-1, keepdim=True) + 2.0**-24 * D * (g * out).abs().sum(-1, keepdim=True)
    dS = P * (dP - delta)
    eds = P * (edp + edelta) + ep * (dP - delta).abs()
    eds = eds * (1 + u) + u * dS.abs() + torch.where(mask, tiny, 0.0)
    shared = lambda x: x.view(B, H // G, G, *x.shape[2:]).sum(2)
    values = [out, scale * dS @ kk, scale * shared(dS.transpose(-1, -2) @ q), shared(P.transpose(-1, -2) @ g)]
    bounds = [eo, scale * eds @ kk.abs(), scale * shared(eds.transpose(-1, -2) @ q.abs()),
              shared(rounded.transpose(-1, -2) @ g.abs())]
    sums = 2.0**-24 * Q * G  # the products' own float32 sums
    size = [None, scale * dS.abs() @ kk.abs(), scale * shared(dS.abs().transpose(-1, -2) @ q.abs()),
            shared(P.transpose(-1, -2) @ g.abs())]
    for i in range(1, 4):
        bounds[i] = bounds[i] + sums * size[i] + u * values[i].abs() + tiny
    return values, bounds


def assert_within(got: torch.Tensor, value: torch.Tensor, bound: torch.Tensor, what: str = ""):
    got = got.detach().cpu().double()
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)} != {tuple(value.shape)}"
    off = (got - value).abs() > bound
    if off.any() or not torch.isfinite(got).all():
        off |= ~torch.isfinite(got)
        i = int(off.reshape(-1).nonzero()[0])
        raise AssertionError(f"{what}: {int(off.sum())} of {got.numel()} out of bounds, first at {i}: got "
                             f"{got.reshape(-1)[i].item()!r}, value {value.reshape(-1)[i].item()!r}, bound "
                             f"{bound.reshape(-1)[i].item()!r}; largest error / bound "
                             f"{((got - value).abs() / bound).max().item():.2f}")
