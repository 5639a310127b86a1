"""The first rows of long sequences see few keys, whatever the window: their dq takes the output's rounding through delta
at nearly full size, unless what the rounding left is kept for them.

Limit 1.75 of the error of a rounded result: the result's own rounding, one of every weight in the output that delta is
formed from (at most as much), and float32 sums: 2 ** 0.5, and room for the keys' common part. Without what the output's
rounding left a third of that size is added, times the output's share of keys whose values do not cancel."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.window_attention import window_attention
from oracle import attention as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 64)],
                         ids=["bf16-128", "bf16-64", "f16-64"])
@pytest.mark.parametrize("window,sinks,starts", [(None, 0, None), (300, 4, None), (None, 0, 301)])
def test_error_of_first_rows(device, dtype, D, window, sinks, starts):
    B, T, H, n = 8, 620, 8, 12
    g = gen(D)
    q, k, v, do = (torch.randn((B, T, H, D), generator=g).to(dtype).transpose(1, 2) for _ in range(4))
    x = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    i = starts or 0
    first = None if starts is None else torch.full((B,), starts, dtype=torch.int32, device=device)
    dq = torch.autograd.grad(window_attention(*x, window=window, sinks=sinks, starts=first), x, do.to(device))[0].cpu()
    torch.cuda.synchronize()
    # causal: the first rows depend on the first tokens alone
    part = [t[:, :, i : i + n] for t in (q, k, v, do)]
    want = ref.attention(*part[:3], ref.masks(B, n, window, sinks), None, part[3])[0][1]
    for rows in (slice(1, 2), slice(2, 4), slice(4, n)):
        e = want[:, :, rows]
        off = (dq[:, :, i : i + n][:, :, rows].double() - e).norm() / (e.to(dtype).double() - e).norm()
        assert off <= 1.75, f"rows {rows.start} to {rows.stop - 1}: {off:.2f} times the error of a rounded result"
