"""Token embedding and its gradient against the formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.token_embedding import TokenEmbedding, token_embedding
from oracle import token_embedding as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ids(gen, n, rows, kind):
    if kind == "even":
        return torch.randint(0, rows, (n,), generator=gen)
    if kind == "text":  # the k-th id about 1 / k of the time
        return (float(rows) ** torch.rand(n, generator=gen, dtype=torch.float64)).long().clamp(1, rows) - 1
    if kind == "one":
        return torch.full((n,), rows // 2)
    if kind == "strange":  # also ids that are no rows
        ids = torch.randint(-3, rows + 3, (n,), generator=gen)
        ids[:: 7] = torch.tensor([-(1 << 40), 1 << 40, (1 << 32) + 1, -1])[torch.arange(len(ids[::7])) % 4]
        return ids
    raise ValueError(kind)


def _check(out, dw, ids, w, grad, scale, padding, what):
    ids, w, grad = ids.cpu(), w.detach().cpu(), grad.cpu()
    want = oracle.embedding(ids, w, scale)
    err = (out.detach().cpu().double() - want).abs()
    assert (err <= oracle.allowed(want, want.abs(), 0, w.dtype)).all(), f"{what}: out off by {err.max()}"
    want, size, terms = oracle.gradient(ids, grad, w.shape[0], scale, padding)
    err = (dw.cpu().double() - want).abs()
    assert (err <= oracle.allowed(want, size, terms[:, None], w.dtype)).all(), f"{what}: dW off by {err.max()}"


CASES = [
    # tokens, rows, dim, kind
    (1, 1, 1, "even"), (1, 7, 8, "even"), (5, 3, 9, "even"), (15, 40, 333, "text"), (17, 300, 64, "strange"),
    (64, 1, 16, "one"), (257, 1000, 8, "one"), (1023, 5, 24, "even"), (1025, 64, 256, "text"), (2049, 17, 72, "strange"),
    (3000, 100, 130, "one"), (5003, 32001, 40, "text"), (4096, 600000, 8, "even"), (4097, 555, 1024, "text"),
    (300, 20, 5000, "text"), (33000, 900, 48, "text"), (40000, 3, 16, "even"),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,rows,dim,kind", CASES)
def test_values_and_gradients(tokens, rows, dim, kind, dtype, device):
    gen = torch.Generator().manual_seed(tokens + rows)
    w = torch.randn((rows, dim), generator=gen).to(dtype).to(device).requires_grad_()
    ids = _ids(gen, tokens, rows, kind).to(device)
    grad = torch.randn((tokens, dim), generator=gen).to(dtype).to(device)
    for wide, scale, padding in ((True, 1.0, None), (False, -1.37, rows // 3)):
        if not wide:
            ids = ids.clamp(-(1 << 31), (1 << 31) - 1).int()
        out = token_embedding(ids, w, scale=scale, padding_idx=padding)
        (dw,) = torch.autograd.grad(out, w, grad)
        assert out.dtype == dw.dtype == dtype and out.shape == (tokens, dim) and dw.shape == w.shape
        _check(out, dw, ids, w, grad, scale, padding, f"wide {wide}")
        (again,) = torch.autograd.grad(token_embedding(ids, w, scale=scale, padding_idx=padding), w, grad)
        assert torch.equal(dw, again)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_strides_and_alignment(dtype, device):
    gen = torch.Generator().manual_seed(3)
    table = torch.randn((50, 96), generator=gen).to(dtype).to(device)
    ids = torch.randint(0, 50, (6, 40), generator=gen).to(device)
    odd = torch.randn(50 * 64 + 1, generator=gen).to(dtype).to(device)
    weights = {"rows apart": table[:, :64], "rows apart, odd": table[:, 3:70], "every second row": table[::2],
               "transposed": torch.randn((64, 50), generator=gen).to(dtype).to(device).T,
               "one row for all": table[:1].expand(50, 96), "not on 16 bytes": odd[1:].view(50, 64)}
    for name, w in weights.items():
        w = w.detach().requires_grad_()
        rows, dim = w.shape
        for what, i in (("whole", ids), ("transposed", ids.T), ("every second", ids[:, ::2])):
            grads = {"whole": torch.randn((*i.shape, dim), generator=gen).to(dtype).to(device),
                     "one for all": torch.randn(dim, generator=gen).to(dtype).to(device).expand(*i.shape, dim),
                     "not on 16 bytes": torch.randn(i.numel() * dim + 1, generator=gen).to(dtype).to(device)[1:].view(*i.shape, dim)}
            for kind, grad in grads.items():
                i_rows = i % rows
                out = token_embedding(i_rows, w, scale=2.0)
                (dw,) = torch.autograd.grad(out, w, grad)
                _check(out, dw, i_rows, w, grad, 2.0, None, f"{name}, ids {what}, gradient {kind}")


def test_empty(device):
    w = torch.randn(5, 8, device=device, requires_grad=True)
    for ids in (torch.zeros(0, dtype=torch.long, device=device), torch.zeros((2, 0, 3), dtype=torch.int32, device=device)):
        out = token_embedding(ids, w)
        assert out.shape == (*ids.shape, 8)
        (dw,) = torch.autograd.grad(out, w, torch.empty_like(out))
        assert torch.equal(dw, torch.zeros_like(w))
    nothing = torch.zeros((0, 8), device=device, requires_grad=True)
    ids = torch.tensor([0, -1, 5], device=device)
    out = token_embedding(ids, nothing)
    assert torch.equal(out, torch.zeros((3, 8), device=device))
    (dw,) = torch.autograd.grad(out, nothing, torch.ones_like(out))
    assert dw.shape == (0, 8)


def test_padding_row_may_hold_anything(device):
    """A padding row is read as any other, and its tokens' gradients (NaN here) go nowhere."""
    w = torch.randn(9, 24, device=device, requires_grad=True)
    ids = torch.tensor([4, 2, 4, 8, 2], device=device)
    grad = torch.ones(5, 24, device=device)
    grad[ids == 2] = float("nan")
    out = token_embedding(ids, w, padding_idx=-7)
    assert torch.equal(out, w[ids])
    (dw,) = torch.autograd.grad(out, w, grad)
    assert torch.equal(dw, torch.zeros_like(w).index_add_(0, ids[ids != 2], grad[ids != 2]))


def test_against_differences(device):
    """The gradient of sum(c * out) by differences of the loss: exact for a linear function up to rounding."""
    gen = torch.Generator().manual_seed(5)
    w = torch.randn((6, 10), generator=gen).to(device).requires_grad_()
    ids = torch.tensor([1, 5, 1, 1, 0], device=device)
    c = torch.randn((5, 10), generator=gen).to(device)
    (dw,) = torch.autograd.grad(token_embedding(ids, w, scale=3.0), w, c)
    loss = lambda x: (token_embedding(ids, x, scale=3.0).double() * c.double()).sum()
    for v, d in ((1, 0), (5, 9), (0, 3), (2, 2)):
        step = torch.zeros_like(w)
        step[v, d] = 0.5
        with torch.no_grad():
            diff = loss(w + step) - loss(w - step)
        # the sums w + step, their products and 50 numbers' double sums: 2^-23 of numbers up to 12 times |c| <= 4, 3 terms
        assert abs(diff.item() - dw[v, d].item()) <= 2**-23 * 12 * 4 * 3 * 2


def test_module_and_other_stream(device):
    e = TokenEmbedding(100, 64, padding_idx=0, scale=8.0, device=device, dtype=BF16)
    ids = torch.randint(0, 100, (4, 50), device=device)
    out = e(ids)
    out.float().sum().backward()
    assert torch.equal(out, e.weight[ids] * 8)  # a power of two: exact
    counts = torch.bincount(ids.flatten(), minlength=100).float()
    counts[0] = 0
    assert torch.equal(e.weight.grad.float(), (counts * 8).to(BF16).float()[:, None].expand(100, 64))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x = token_embedding(ids, e.weight, scale=8.0)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(x, out)


def test_captured(device):
    """Forward and backward in a graph; ids, table and gradient change between replays."""
    gen = torch.Generator().manual_seed(9)
    w = torch.randn((300, 72), generator=gen).to(BF16).to(device).requires_grad_()
    ids = torch.zeros(500, dtype=torch.long, device=device)
    grad = torch.zeros((500, 72), dtype=BF16, device=device)

    def both():
        out = token_embedding(ids, w, scale=0.5, padding_idx=7)
        return out.detach(), torch.autograd.grad(out, w, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = both()
    for kind in ("text", "one", "even", "strange"):
        ids.copy_(_ids(gen, 500, 300, kind))
        grad.copy_(torch.randn((500, 72), generator=gen))
        with torch.no_grad():
            w.copy_(torch.randn((300, 72), generator=gen))
        graph.replay()
        want = both()
        assert torch.equal(out, want[0]) and torch.equal(dw, want[1]), kind


def test_offsets_past_32_bits(device):
    """A table of more than 2^32 bytes and 2^31 numbers: rows at both ends."""
    rows, dim = (1 << 21) + 3, 1032
    w = torch.zeros((rows, dim), dtype=BF16, device=device)
    ids = torch.tensor([0, rows - 1, rows - 1, rows // 2], device=device)
    w[ids] = torch.arange(4, device=device, dtype=BF16)[[0, 2, 2, 3]][:, None]
    w.requires_grad_()
    out = token_embedding(ids, w)
    assert torch.equal(out.float(), torch.tensor([0.0, 2, 2, 3], device=device)[:, None].expand(4, dim))
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw[0].eq(1).all() and dw[rows - 1].eq(2).all() and dw[rows // 2].eq(1).all()
    assert dw.float().sum().item() == 4 * dim
