"""Window attention's float16 gradients hold their precision whatever the size of grad_out: 2-norm of the error of dq,
dk and dv against 64 bits, in units of what rounding the exact result to float16 leaves.

Limit 2: beside the result's own rounding, each gradient takes one rounding of every weight (dv) or of every dS (dk),
and delta takes one of the output (dq, dk); each of these three adds at most as much as the result's rounding for
random inputs, so the root of their squares stays below 3 ** 0.5, and float32 sums are far below."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.window_attention import window_attention
from oracle import attention as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _error(got, exact):
    """2-norm of the error over that of the rounded exact result, where the latter is finite."""
    rounded = exact.to(F16)
    fine = torch.isfinite(rounded)
    assert fine.float().mean() > 0.99 and torch.isfinite(got.cpu()[fine]).all()
    off = lambda x: (x.cpu().double() - exact)[fine].norm()
    return (off(got) / off(rounded)).item()


def _gradients(q, k, v, do, mask):
    """dq, dk, dv in 64 bits."""
    G, scale = q.shape[1] // k.shape[1], q.shape[-1] ** -0.5
    q, do = q.double(), do.double()
    kk, vv = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    P = torch.softmax(torch.where(mask, q @ kk.transpose(-1, -2) * scale, -torch.inf), -1)
    dP = do @ vv.transpose(-1, -2)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    shared = lambda x: x.unflatten(1, (-1, G)).sum(2)
    return scale * dS @ kk, scale * shared(dS.transpose(-1, -2) @ q), shared(P.transpose(-1, -2) @ do)


@pytest.mark.parametrize("D,T,window,sinks", [(64, 2048, None, 0), (128, 2048, None, 0), (64, 2100, 400, 4), (128, 1900, 300, 40)])
@pytest.mark.parametrize("size", [2.0**-12, 1e-3, 1.0, 2.0**13])
def test_error_of_any_size_of_gradients(device, D, T, window, sinks, size):
    g = gen(T + D)
    q, k, v, do = (torch.randn((1, T, h, D), generator=g).transpose(1, 2) for h in (2, 1, 1, 2))
    q, k, v, do = q.to(F16), (k + torch.randn((1, 1, 1, D), generator=g) / 2).to(F16), v.to(F16), (do * size).to(F16)
    x = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*x, window=window, sinks=sinks), x, do.to(device))
    torch.cuda.synchronize()
    want = _gradients(q, k, v, do, ref.masks(1, T, window, sinks))
    for name, a, e in zip(("dq", "dk", "dv"), got, want):
        ratio = _error(a, e)
        assert ratio <= 2, f"{name}: {ratio:.2f} times the error of a rounded result"


def test_rows_of_very_different_sizes(device):
    """Rows of grad_out between 2^-20 and 2^10, mixed: every row of dq keeps its own precision, and dk and dv theirs."""
    T, D = 1500, 64
    g = gen(3)
    q, k, v, do = (torch.randn((1, 1, T, D), generator=g) for _ in range(4))
    do = do * torch.exp2(torch.randint(-20, 11, (1, 1, T, 1), generator=g).float())
    q, k, v, do = (t.to(F16) for t in (q, k, v, do))
    x = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*x), x, do.to(device))
    torch.cuda.synchronize()
    want = _gradients(q, k, v, do, ref.masks(1, T, None, 0))
    for name, a, e in zip(("dq", "dk", "dv"), got, want):
        assert _error(a, e) <= 2, name
    # rows by their size: each size's error on its own
    size = do.double().abs().amax(-1)[0, 0].log2().round()
    for s in size.unique():
        rows = size == s
        if rows.sum() >= 20:
            assert _error(got[0][:, :, rows.to(device)], want[0][:, :, rows]) <= 2, f"rows of 2^{int(s)}"


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_whose_steps_pass_float16(device, D):
    """dS up to 2^18 in the first rows of many short sequences, whose dq, dk and dv a float16 still holds."""
    g = gen(D)
    q, k, v, do = (torch.randn((8, 8, 24, D), generator=g) for _ in range(4))
    q, k, v, do = (q / 4).to(F16), (k / 4).to(F16), (v * 4).to(F16), (do * 2.0**13).clamp(-60000, 60000).to(F16)
    x = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*x), x, do.to(device))
    torch.cuda.synchronize()
    for name, a, e in zip(("dq", "dk", "dv"), got, _gradients(q, k, v, do, ref.masks(1, 24, None, 0))):
        assert _error(a, e) <= 2, name


def test_long_sequences_of_float16(device):
    """Weights of 1 / 16384 are below float16's normal numbers: dv of the late keys keeps its precision."""
    T, D = 16384, 64
    g = gen(8)
    q, k, v, do = (torch.randn((1, T, 1, D), generator=g).transpose(1, 2).to(F16) for _ in range(4))
    do[:, :, : T - 64] = 0  # the last rows' gradients alone
    x = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*x), x, do.to(device))
    torch.cuda.synchronize()
    rows = slice(T - 64, T)
    mask = ref.visible(T, 0, T, None, 0)[rows]
    qq, kk, vv, dd = (t[0, 0].double() for t in (q[:, :, rows], k, v, do[:, :, rows]))
    P = torch.softmax(torch.where(mask, qq @ kk.T / 8, -torch.inf), -1)
    dP = dd @ vv.T
    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) / 8
    for name, a, e in zip(("dq", "dk", "dv"), (got[0][0, 0, rows], got[1][0, 0], got[2][0, 0]), (dS @ kk, dS.T @ qq, P.T @ dd)):
        assert _error(a, e) <= 2, name
