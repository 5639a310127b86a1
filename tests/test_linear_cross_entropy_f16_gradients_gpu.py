"""Cross entropy of a linear layer in float16, its tokens' gradients far apart in size."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.linear_cross_entropy import linear_cross_entropy
from oracle import linear_cross_entropy as oracle

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _near(got, want, bound, what):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(err / bound).max():.2f} of its bound"


def _inputs(n, V, D, seed, device):
    """Rows of weight with a common part, which only the softmax's sum over all of them gives dx; losses' gradients of
    either sign from 2^-14 to 2^10, a few of them 0."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn((V, D), generator=gen) * 0.64 * D**-0.5
    w += 2 * w.std() * torch.randn(D, generator=gen)
    x = torch.randn((n, D), generator=gen)
    labels = torch.randint(0, V, (n,), generator=gen)
    grad = torch.exp2(10 - 24 * torch.rand(n, generator=gen)) * (torch.randint(0, 2, (n,), generator=gen) * 2 - 1)
    grad[::17] = 0
    labels[5::11] = -100
    return x.to(F16).to(device).requires_grad_(), w.to(F16).to(device).requires_grad_(), labels.to(device), grad


@pytest.mark.parametrize("n,V,D", [(60, 32000, 64), (200, 500, 64), (300, 32000, 72), (1000, 200, 40), (3, 7, 5)])
def test_gradients_far_apart(n, V, D, device):
    """Every token's row of dx is as precise as alone, whatever the other tokens' gradients are."""
    x, w, labels, grad = _inputs(n, V, D, n + V, device)
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), grad.to(device), retain_graph=True)
    values, bounds = oracle.loss_and_gradients(x.detach().cpu(), w.detach().cpu(), labels.cpu(), -100, "none", grad.double(),
                                               each=True)
    for name, got, want, bound in zip(("dx", "dW"), (dx, dw), values[1:], bounds[1:]):
        _near(got, want, bound, name)
    assert not dx[::17].any()
    again = torch.autograd.grad(loss, (x, w), grad.to(device))  # nothing is used up
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("size", [2.0**-18, 2.0**-4, 1.0, 2.0**6])
def test_hidden_states_of_any_size(size, device):
    """The tokens' powers of two go to a copy of the hidden states for dW: states of any size leave it room."""
    x, w, labels, grad = _inputs(300, 700, 64, 1, device)
    with torch.no_grad():
        x *= size
        x[7] *= 2.0**6
    grad = grad / 2.0**10
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    got = torch.autograd.grad(loss, (x, w), grad.to(device))
    values, bounds = oracle.loss_and_gradients(x.detach().cpu(), w.detach().cpu(), labels.cpu(), -100, "none", grad.double(),
                                               each=True)
    for name, g, want, bound in zip(("dx", "dW"), got, values[1:], bounds[1:]):
        _near(g, want, bound, name)


def test_what_is_not_a_number(device):
    """A gradient that is infinite or NaN spoils its own row of dx (and dW), not the others'."""
    x, w, labels, grad = _inputs(300, 700, 64, 2, device)
    keep = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="none"), x, grad.to(device))[0]
    for odd in (float("inf"), float("nan")):
        some = grad.clone()
        some[3] = odd
        dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="none"), (x, w), some.to(device))
        spoilt = (~dx.isfinite()).any(1).nonzero().flatten().tolist()
        assert spoilt == [3] and not dw.isfinite().all()
        assert torch.equal(dx[:3], keep[:3]) and torch.equal(dx[4:], keep[4:])
