"""Cross entropy of a linear layer under torch.autocast: as a linear layer there, in autocast's type."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.linear_cross_entropy import linear_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("hidden", [torch.float32, torch.bfloat16, torch.float16], ids=["h32", "hb16", "h16"])
def test_autocast(hidden, dtype, device):
    """A float32 table and states of any of the types: autocast's type is what the operator sees, and gradients come back
    in the tensors' own."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn((2, 70, 40), generator=gen).to(hidden).to(device).requires_grad_()
    w = (torch.randn((300, 40), generator=gen) / 4).to(device).requires_grad_()
    labels = torch.randint(0, 300, (2, 70), generator=gen).to(device)
    with torch.autocast("cuda", dtype=dtype):
        loss = linear_cross_entropy(x, w, labels)
        with torch.no_grad():
            assert torch.equal(linear_cross_entropy(x, w, labels), loss)
    got = torch.autograd.grad(loss, (x, w))
    x2, w2 = (t.detach().to(dtype).requires_grad_() for t in (x, w))
    want = linear_cross_entropy(x2, w2, labels)
    assert torch.equal(loss, want)
    for g, t, g2 in zip(got, (x, w), torch.autograd.grad(want, (x2, w2))):
        assert g.dtype == t.dtype and torch.equal(g, g2.to(t.dtype))
    with torch.autocast("cuda", dtype=dtype, enabled=False), pytest.raises(NotImplementedError):
        linear_cross_entropy(x, w, labels)
