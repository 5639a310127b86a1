"""How far the gradients of the cross entropy of a linear layer lie from 64 bits, over what rounding the exact ones to the
inputs' type once leaves (2-norms)."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.linear_cross_entropy import linear_cross_entropy

pytestmark = pytest.mark.gpu


def _ratios(n, V, D, dtype, device):
    gen = torch.Generator().manual_seed(n + V)
    w = torch.randn((V, D), generator=gen) * 0.64 * D**-0.5
    labels = torch.randint(0, V, (n,), generator=gen)
    x = torch.randn((n, D), generator=gen) + 12 * torch.rand((n, 1), generator=gen) * w[labels] / w[labels].square().sum(1, keepdim=True)
    x, w, labels = x.to(dtype).to(device).requires_grad_(), w.to(dtype).to(device).requires_grad_(), labels.to(device)
    got = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="sum"), (x, w))
    xx, ww = x.detach().double(), w.detach().double()
    d = (xx @ ww.T).softmax(1)
    d[torch.arange(n, device=device), labels] -= 1
    return [((g.double() - e).norm() / (e.to(dtype).double() - e).norm()).item() for g, e in zip(got, (d @ ww, d.T @ xx))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n,V,D", [(129, 300, 64), (300, 5000, 512), (2048, 256, 256), (1800, 20011, 200)])
def test_more_than_128_tokens(n, V, D, dtype, device):
    """The logits' gradients are rounded once for the products: independent errors of relative size r in terms that are
    independent too add r to a result of relative error r of its own, sqrt(2) in all; 5 % for what these draws differ by."""
    dx, dw = _ratios(n, V, D, dtype, device)
    assert dx <= 1.05 * 2**0.5 and dw <= 1.05 * 2**0.5, (dx, dw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n,V,D", [(1, 300, 64), (64, 20011, 512), (128, 256, 256)])
def test_up_to_128_tokens(n, V, D, dtype, device):
    """They enter as two numbers, off by 2^-16 of themselves at most (2^-8 of a bf16's 2^-8): 2^-16 / 2^-9 of a result's own
    rounding. float32 sums of up to 512 terms: 2^-24 sqrt(512) / 2^-12 in f16, 0.6 %."""
    dx, dw = _ratios(n, V, D, dtype, device)
    assert dx <= 1.02 and dw <= 1.02, (dx, dw)
