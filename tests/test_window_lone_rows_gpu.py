"""Window attention's gradients where a query sees one key alone: its weight is 1 whatever q and k are, so dq of the
row and what the row gives to dk are 0, exactly."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.window_attention import window_attention
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64)]
TYPE_IDS = ["bf16-128", "bf16-64", "f16-128", "f16-64"]


def _run(device, B, T, H, Hk, D, dtype, seed, spoil=None, **kw):
    g = gen(seed)
    q, k, v, do = (torch.randn((B, T, h, D), generator=g).to(dtype).transpose(1, 2).to(device) for h in (H, Hk, Hk, H))
    if spoil is not None:
        do[spoil] = float("nan")
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    for name in ("starts", "ends"):
        if name in kw:
            kw[name] = torch.tensor(kw[name], dtype=torch.int32, device=device)
    out = window_attention(*x, **kw)
    grads = torch.autograd.grad(out, x, do)
    torch.cuda.synchronize()
    return [t.detach().cpu() for t in (v, do, out, *grads)]


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("B,T,H,Hk,kw", [
    (3, 1, 4, 2, {}), (1, 1, 3, 3, dict(window=5, sinks=2)), (2, 200, 4, 1, dict(window=1)), (1, 33, 2, 2, dict(window=1)),
    (3, 150, 4, 2, dict(starts=[149, 31, 64], ends=[150, 32, 65])),  # one token of padded batches
], ids=["one-token", "one-token-window", "window-1", "window-1-short", "one-token-padded"])
def test_every_row_is_alone(device, dtype, D, B, T, H, Hk, kw):
    v, do, out, dq, dk, dv = _run(device, B, T, H, Hk, D, dtype, T, **kw)
    assert (dq == 0).all() and (dk == 0).all()
    starts, ends = kw.get("starts", [0] * B), kw.get("ends", [T] * B)
    for b in range(B):  # out is v and dv the group's sum of grad_out
        i, j = int(starts[b]), int(ends[b])
        assert torch.equal(out[b, :, i:j], v[b, :, i:j].repeat_interleave(H // Hk, 0))
        want = do[b, :, i:j].double().unflatten(0, (Hk, H // Hk)).sum(1)
        terms = do[b, :, i:j].double().abs().unflatten(0, (Hk, H // Hk)).sum(1)
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-20 * terms
        assert ((dv[b, :, i:j].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("starts", [0, 31, 45])
def test_the_first_row_is_alone(device, dtype, D, starts):
    """A grad_out that is 0 but at each sequence's first row: nothing but dv of that row."""
    B, T, H, Hk = 2, 90, 4, 2
    g = gen(starts)
    q, k, v, do = (torch.randn((B, h, T, D), generator=g).to(dtype).to(device) for h in (H, Hk, Hk, H))
    only = torch.zeros_like(do)
    only[:, :, starts] = do[:, :, starts]
    x = [t.requires_grad_(True) for t in (q, k, v)]
    first = torch.full((B,), starts, dtype=torch.int32, device=device)
    for window, sinks in ((None, 0), (20, 3)):
        dq, dk, dv = torch.autograd.grad(window_attention(*x, window=window, sinks=sinks, starts=first), x, only)
        full = torch.autograd.grad(window_attention(*x, window=window, sinks=sinks, starts=first), x, do)
        torch.cuda.synchronize()
        assert (dq == 0).all() and (dk == 0).all() and (dv[:, :, starts] != 0).any()
        assert (full[0][:, :, starts] == 0).all() and (full[0][:, :, starts + 1] != 0).any()


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
def test_nan_of_a_lone_row_is_not_hidden(device, dtype, D):
    """A NaN in grad_out of a lone row stays one in its dq and in its key's dk, as in the formulas."""
    _, _, _, dq, dk, dv = _run(device, 2, 1, 2, 1, D, dtype, 5, spoil=(0, 1, 0, 3))
    assert dq[0, 1].isnan().all() and dk[0].isnan().all() and dv[0, 0, 0, 3].isnan()
    assert (dq[1] == 0).all() and (dq[0, 0] == 0).all() and (dk[1] == 0).all()
