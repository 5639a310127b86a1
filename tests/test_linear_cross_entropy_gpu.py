"""Cross entropy of a linear layer against the formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

from modelos_amd import _lib
from modelos_amd.linear_cross_entropy import linear_cross_entropy
from oracle import linear_cross_entropy as oracle

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _inputs(n, V, D, dtype, device, seed=0, lean=12.0, ignored=0.0):
    """Normed hidden states that lean towards their label's row; labels in [0, V), -100 for the ignored."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn((V, D), generator=gen) * 0.64 * D**-0.5
    labels = torch.randint(0, V, (n,), generator=gen)
    x = torch.randn((n, D), generator=gen)
    x += lean * torch.rand((n, 1), generator=gen) * w[labels] / w[labels].square().sum(1, keepdim=True).clamp_min(1e-6)
    labels[torch.rand(n, generator=gen) < ignored] = -100
    return x.to(dtype).to(device).requires_grad_(), w.to(dtype).to(device).requires_grad_(), labels.to(device), gen


def _near(got, want, bound, what):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(err / bound.clamp_min(1e-300)).max():.2f} of its bound"


def _both(x, w, labels, reduction, gen, size=1.0, **options):
    loss = linear_cross_entropy(x, w, labels, reduction=reduction, **options)
    grad = torch.full((), size) if reduction != "none" else size * torch.rand(labels.shape, generator=gen)
    grads = torch.autograd.grad(loss, (x, w), grad.to(x.device))
    return loss, grad, grads


def _check(x, w, labels, reduction, gen, size=1.0, ignore_index=-100):
    loss, grad, grads = _both(x, w, labels, reduction, gen, size, ignore_index=ignore_index)
    assert loss.dtype == torch.float32 and loss.shape == (labels.shape if reduction == "none" else ())
    assert all(g.shape == t.shape and g.dtype == t.dtype for g, t in zip(grads, (x, w)))
    D = x.shape[-1]
    values, bounds = oracle.loss_and_gradients(x.detach().cpu().reshape(-1, D), w.detach().cpu(), labels.cpu().reshape(-1),
                                               ignore_index, reduction, grad.double().reshape(-1) if reduction == "none" else grad.double())
    for name, got, want, bound in zip(("loss", "dx", "dW"), (loss, *grads), values, bounds):
        _near(got.reshape(want.shape), want, bound, f"{name}, {reduction}")
    return loss, grads


SIZES = [
    # tokens, vocab, dim
    (1, 1, 8), (1, 2, 1), (3, 7, 5), (64, 300, 64), (255, 257, 72), (257, 130, 200), (256, 256, 256), (300, 1000, 333),
    (31, 5000, 1000), (1000, 513, 264), (17, 20011, 128), (700, 40, 512),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,V,D", SIZES)
def test_values_and_gradients(n, V, D, reduction, dtype, device):
    x, w, labels, gen = _inputs(n, V, D, dtype, device, n + V, ignored=0.3 if n > 100 else 0.0)
    _check(x, w, labels, reduction, gen)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_several_pieces(dtype, device):
    """Few tokens and much vocabulary, whose last tile is not full."""
    x, w, labels, gen = _inputs(70, 2 * 16384 + 16300, 64, dtype, device)
    labels[:4] = torch.tensor([16383, 16384, 32768, 2 * 16384 + 16299])
    _check(x, w, labels, "mean", gen)


@pytest.mark.parametrize("dtype,size", [(BF16, 2.0**-40), (BF16, 2.0**20), (F16, 2.0**-10), (F16, 2.0**10)])
def test_gradients_of_any_size(dtype, size, device):
    """Softmax weights of 500 entries times 2^-10 lie below f16's smallest numbers: results in its range keep their precision."""
    x, w, labels, gen = _inputs(200, 500, 64, dtype, device, lean=0.0)
    _check(x, w, labels, "none", gen, size)


def test_large_logits(device):
    """A label far below the largest logit: the sum of the exponentials leaves float32 against the label's."""
    x, w, labels, gen = _inputs(100, 700, 64, BF16, device, lean=0.0)
    with torch.no_grad():
        x[::3] *= 200
        x[1::3] *= 20
    loss, _ = _check(x, w, labels, "none", gen)
    assert loss.max() > 200


def test_rows_that_lean_all_one_way(device):
    """weight with a common part, which d (whose sum over the vocabulary is 0) cancels."""
    x, w, labels, gen = _inputs(200, 3000, 128, BF16, device)
    with torch.no_grad():
        w += w.std() * 2 * torch.randn(128, generator=gen).to(device)
    _check(x, w, labels, "mean", gen)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_nothing_counts(reduction, device):
    x, w, labels, gen = _inputs(70, 90, 40, BF16, device)
    with torch.no_grad():
        x.fill_(float("nan"))
    for some in (torch.full_like(labels, -100), torch.full_like(labels, 90), labels - 1000):
        loss, _, (dx, dw) = _both(x, w, some, reduction, gen)
        assert not loss.any() and not dx.any() and not dw.any()
    x = torch.zeros((0, 40), dtype=BF16, device=device, requires_grad=True)
    loss, _, (dx, dw) = _both(x, w, labels[:0], reduction, gen)
    assert not loss.any() and dx.shape == (0, 40) and not dw.any()


def test_what_ignored_tokens_hold(device):
    x, w, labels, gen = _inputs(300, 200, 64, BF16, device, ignored=0.4)
    labels[7], labels[9] = 200, -1  # outside
    with torch.no_grad():
        away = (labels < 0) | (labels >= 200)
        x[away] = torch.tensor([float("nan"), float("inf")], device=device, dtype=BF16)[torch.arange(int(away.sum())) % 2][:, None]
    for ignore in (-100, 3):
        _check(x.detach().requires_grad_(), w, labels.where(labels != -100, ignore), "none", gen, ignore_index=ignore)
        labels = labels.where(labels != 3, 4)


def test_a_token_that_is_not_a_number(device):
    """Its loss and its gradient are NaN, and dW's rows; the other tokens' losses and gradients are not."""
    x, w, labels, gen = _inputs(300, 200, 64, BF16, device)
    with torch.no_grad():
        x[11, 5] = float("nan")
    loss, _, (dx, dw) = _both(x, w, labels, "none", gen)
    assert loss.isnan().nonzero().tolist() == [[11]] and dw.isnan().all()
    assert dx.isnan().any(1).nonzero().tolist() == [[11]]


def test_strides(device):
    """Rows apart, transposed, not on 16 bytes, one for all; labels of 32 bits and of strides; shapes of several axes."""
    _, w0, labels, gen = _inputs(120, 150, 64, BF16, device)
    wide = torch.randn((6, 20, 2, 64), generator=gen).to(BF16).to(device)
    odd = torch.randn(120 * 64 + 1, generator=gen).to(BF16).to(device)
    hidden = {"rows apart": wide[:, :, 1], "transposed": wide[:, :, 0].transpose(0, 1), "odd": odd[1:].view(6, 20, 64),
              "one for all": wide[0, 0, 0].expand(6, 20, 64), "columns apart": wide.flatten()[: 6 * 20 * 128].view(6, 20, 128)[..., ::2]}
    weights = {"rows apart": torch.cat([w0, w0], 1)[:, :64], "odd": torch.cat([w0.flatten()[:1], w0.flatten()])[1:].view(150, 64),
               "transposed": w0.T.contiguous().T, "one for all": w0[:1].expand(150, 64), "whole": w0}
    for name, x in hidden.items():
        for kind, w in weights.items():
            y = labels.view(*x.shape[:-1])
            y = y.int() if kind == "odd" else torch.stack([y, y], -1)[..., 0]
            _check(x.detach().requires_grad_(), w.detach().requires_grad_(), y, "mean", gen)
    x = wide[0, 0, 0].detach().requires_grad_()  # a single token without an axis of its own
    _check(x, w0, labels[0], "mean", gen)


def test_one_gradient_alone(device):
    x, w, labels, gen = _inputs(300, 700, 136, BF16, device)
    loss, grad, (dx, dw) = _both(x, w, labels, "mean", gen)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, w.detach(), labels), x)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x.detach(), w, labels), w)[0], dw)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, labels), loss)
    loss = linear_cross_entropy(x, w, labels)  # twice through one graph, with the same bits
    for _ in range(2):
        again = torch.autograd.grad(loss, (x, w), retain_graph=True)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_against_differences(device):
    """d loss / d w along one direction, by differences of losses with weights moved along it: exact in bf16, as the step is
    a power of two of numbers with few digits."""
    gen = torch.Generator().manual_seed(3)
    w = (torch.randint(-8, 9, (50, 32), generator=gen) / 16).to(BF16).to(device).requires_grad_()
    x = (torch.randint(-8, 9, (40, 32), generator=gen) / 8).to(BF16).to(device).requires_grad_()
    labels = torch.randint(0, 50, (40,), generator=gen).to(device)
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="sum"), (x, w))
    h = 2.0**-6
    for t, grad in ((w, dw), (x, dx)):
        to = torch.randint(-1, 2, t.shape, generator=gen).to(BF16).to(device)
        with torch.no_grad():
            t0 = t.clone()
            ends = []
            for s in (h, -h):
                t.copy_(t0 + s * to)
                assert torch.equal(t.double(), t0.double() + s * to.double())
                ends.append(linear_cross_entropy(x, w, labels, reduction="none").double().sum())
            t.copy_(t0)
        slope = (ends[0] - ends[1]).item() / (2 * h)
        exact = (grad.double() * to.double()).sum().item()
        # third derivative: h^2 / 6 of 40 tokens' softmax moments, logits' slopes up to 32 x 1: (32)^3; measured against
        # the slopes' own spread |x to| <= 8 typically: 40 h^2 / 6 * 8^3; float32 losses of 4 each, 2^-22 / h; bf16 results
        bound = 40 * h * h / 6 * 512 + 40 * 4 * 2.0**-22 / h + 2.0**-8 * (grad.double().abs() * to.double().abs()).sum().item()
        assert abs(slope - exact) <= bound


def test_captured(device):
    """Forward and backward in a graph: hidden states, weights, labels (and how many count) change between replays."""
    x, w, labels, gen = _inputs(300, 600, 72, BF16, device)
    grad = torch.ones((), device=device)

    def both():
        loss = linear_cross_entropy(x, w, labels)
        return loss.detach(), *torch.autograd.grad(loss, (x, w), grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k, ignored in enumerate((0.0, 0.9, 1.0, 0.3)):
        x2, w2, labels2, _ = _inputs(300, 600, 72, BF16, device, seed=k, ignored=ignored)
        with torch.no_grad():
            x.copy_(x2)
            w.copy_(w2)
        labels.copy_(labels2)
        grad.fill_(2.0**k)
        graph.replay()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_other_stream(device):
    x, w, labels, gen = _inputs(100, 600, 64, BF16, device)
    want = _both(x, w, labels, "mean", gen)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _both(x, w, labels, "mean", gen)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


def test_few_of_many_tokens_count(device):
    """dW's sum over 3000 tokens is split (one result of 256 x 256); with a handful that count most splits have nothing."""
    x, w, labels, gen = _inputs(3000, 200, 64, BF16, device)
    for n in (0, 1, 65, 200, 2999, 3000):
        some = labels.clone()
        some[torch.randperm(3000, generator=gen)[: 3000 - n].to(device)] = -100
        _check(x, w, some, "mean", gen)


@pytest.mark.parametrize("n", [60, 300])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_losses_near_nothing(n, dtype, device):
    """Sure tokens: losses of 1e-2 down to 1e-11 and their gradients keep their precision. log(1 + s) of a small s is off
    by as much of itself as s is, and s by the logits' errors."""
    x, w, labels, gen = _inputs(n, 400, 64, dtype, device, lean=0.0)
    with torch.no_grad():
        far = torch.linspace(10, 40, n)[:, None].to(device) * w[labels].float()
        x += (far / w[labels].float().square().sum(1, keepdim=True)).to(dtype)
    loss, grad, (dx, dw) = _both(x, w, labels, "none", gen)
    xx, ww = x.detach().cpu().double(), w.detach().cpu().double()
    logits = xx @ ww.T
    y = labels.cpu()[:, None]
    others = (logits - logits.gather(1, y)).scatter(1, y, -float("inf"))
    want = torch.log1p(others.exp().sum(1))
    assert want.min() < 1e-10 and want.max() > 1e-3  # what the inputs are
    # two logits of D products each, their difference and its exponential, the sums
    e = 2.0**-24 * (2 * (64 + 2) * (xx.abs() @ ww.abs().T).max(1).values + 8 * others[others > -1e9].abs().max() + 60)
    assert ((loss.cpu().double() - want).abs() <= e * want).all()
    g = grad.double()[:, None]
    p = others.exp() / (1 + others.exp().sum(1, keepdim=True))
    d = torch.where(torch.arange(400) == y, torch.expm1(-want)[:, None], p) * g
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    # f16: the smallest of d, 2^-24 below 2^14 times the largest gradient
    lost = 2.0**-38 * g.abs().max() if dtype == F16 else 0.0
    for got, exact, size in ((dx, d @ ww, d.abs() @ ww.abs()), (dw, d.T @ xx, d.T.abs() @ xx.abs())):
        other = (torch.ones_like(d) @ ww.abs() if got is dx else torch.ones_like(d).T @ xx.abs()) * lost
        bound = (u + 4 * e.max() + 2.0**-17) * size + other + u * exact.abs() + tiny
        assert ((got.cpu().double() - exact).abs() <= bound).all()


def test_offsets_past_32_bits(device):
    """A weight of more than 2^32 bytes and 2^31 numbers, all zeros but for three rows at its ends and in the middle."""
    V, D = (1 << 21) + 5, 1032
    w = torch.zeros((V, D), dtype=BF16, device=device)
    rows = torch.tensor([0, V // 2, V - 1], device=device)
    w[rows] = torch.tensor([1.0, 2.0, -1.0], device=device, dtype=BF16)[:, None] / 64
    w.requires_grad_()
    x = (torch.eye(3, D, device=device) * 64).to(BF16).requires_grad_()  # the logits of a token: 1, 2 and -1 at the three rows
    labels = rows[[1, 2, 0]]
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    total = torch.tensor([1.0, 2.0, -1.0]).double().exp().sum() + V - 3
    want = total.log() - torch.tensor([2.0, -1.0, 1.0]).double()
    assert ((loss.cpu().double() - want).abs() <= 2.0**-20 * want).all()
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    p = torch.tensor([1.0, 2.0, -1.0]).double().exp() / total
    for k, v in enumerate(rows.tolist()):  # column t of row v: the d of token t times its 64
        d = p[k] - (labels.cpu() == v).double()
        assert ((dw[v, :3].cpu().double() - 64 * d).abs() <= 2.0**-7 * 64 * d.abs()).all()
        assert not dw[v, 3:].any()
    other = dw[[1, V // 2 - 1, V // 2 + 1, V - 2], :3].cpu().double()
    assert ((other - 64 / total).abs() <= 2.0**-7 * 64 / total).all()
    exact = (p[None] - (labels.cpu()[:, None] == rows.cpu()[None]).double()) @ torch.tensor([1.0, 2.0, -1.0]).double() / 64
    assert ((dx.cpu().double() - exact[:, None]).abs() <= 2.0**-7 * exact[:, None].abs()).all()


@pytest.mark.parametrize("ignored", [0.3, 0.999])
@pytest.mark.parametrize("V", [16384 + 300, 2 * 16384 + 1])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_pieces_of_many_tokens(dtype, V, ignored, device):
    """24600 tokens: the backward takes 64 tiles of the vocabulary at a time or fewer. The oracle's 64-bit products on the GPU."""
    n, D = 24600, 24
    x, w, labels, gen = _inputs(n, V, D, dtype, device, V, ignored=ignored)
    labels[:6] = torch.tensor([0, 16383, 16384, V // 2 // 256 * 256, V - 2, V - 1])
    assert _lib.load().pkm_linear_ce_bwd_workspace_size(n, V, D) < 24832 * 2 * V * 0.7  # not all of d
    loss, grad, grads = _both(x, w, labels, "mean", gen)
    values, bounds = oracle.loss_and_gradients(x.detach(), w.detach(), labels, -100, "mean", grad.double().to(device))
    for name, got, want, bound in zip(("loss", "dx", "dW"), (loss, *grads), values, bounds):
        _near(got, want.cpu(), bound.cpu(), name)


@pytest.mark.parametrize("n", [3, 200])
def test_infinite_logits(n, device):
    """Logits of -infinity: no part of a loss, but of the token whose label has it, whose loss is infinite."""
    w = torch.zeros((3, 64), dtype=BF16, device=device)
    w[:, 0] = torch.tensor([-float("inf"), 0.0, 1.0])
    x = torch.eye(1, 64, dtype=BF16, device=device).expand(n, 64)
    labels = torch.arange(n, device=device) % 3
    loss = linear_cross_entropy(x, w, labels, reduction="none").cpu().double()
    want = torch.nn.functional.cross_entropy((x @ w.T).cpu().double(), labels.cpu(), reduction="none")
    assert torch.equal(torch.isinf(loss), labels.cpu() == 0) and not loss.isnan().any()
    fine = labels.cpu() != 0
    assert ((loss - want)[fine].abs() <= 2.0**-21 * want[fine]).all()


@pytest.mark.parametrize("n", [64, 300])
@pytest.mark.parametrize("V", [40000, 151936, 200003])
def test_a_flat_vocabulary_far_above_the_labels(V, n, device):
    """Labels 60 to 100 below a vocabulary of equal logits: the sums of the parts of the vocabulary, each against the
    label's logit, stay in float32 one by one before all of them together do. Every logit is exact: -gap in a label's
    column 0, zeros elsewhere, a 1 in column 1 of the other rows for dx to see the softmax."""
    gap = torch.linspace(60, 100, n).to(BF16)
    labels = torch.randperm(V, generator=torch.Generator().manual_seed(V + n))[:n]
    w = torch.zeros((V, 8), dtype=BF16)
    w[:, 1] = 1
    w[labels, 0], w[labels, 1] = -gap, 0
    x = torch.eye(1, 8, dtype=BF16).expand(n, 8).contiguous().to(device).requires_grad_()
    w = w.to(device).requires_grad_()
    loss = linear_cross_entropy(x, w, labels.to(device), reduction="none")
    dx, dw = (g.cpu().double() for g in torch.autograd.grad(loss.sum(), (x, w)))
    gap = gap.double()
    total = V - n + (-gap).exp().sum()
    want = total.log() + gap
    # the exponent's rounding at up to 100 log2(e), the sum of V exponentials, the logarithm's and the sums' roundings
    bound = 2.0**-24 * (4 * gap + 4 * total.log() + 2 * V**0.5 + 16)
    _near(loss, want, bound, "loss")
    # d is rounded, all entries' alike, and the results are; exp(l - lse) is off by what lse is
    off = 2 * 2.0**-8 + 2.0**-16 + 2 * bound.max()
    p = 1 / total
    _near(dx[:, 1], ((V - n) * p).expand(n), off, "dx from the softmax")
    _near(dx[:, 0], gap, off * gap, "dx from the label")
    others = torch.ones(V, dtype=torch.bool)
    others[labels] = False
    _near(dw[others, 0], (n * p).expand(V - n), off * n * p, "dW of the others")
    _near(dw[labels, 0], -torch.ones(n), off + 1e-20, "dW of the labels")
    assert not dw[:, 1:].any()


@pytest.mark.parametrize("n", [12288, 12289, 70001, (1 << 20) + 5])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 0.9999])
def test_long_batches(ignored, kind, n, device):
    """From 12289 tokens on the kept ones are counted by a launch of its own. The oracle's 64-bit products on the GPU."""
    x, w, labels, gen = _inputs(n, 40, 16, BF16, device, n, lean=4.0, ignored=ignored)
    labels[n - 1] = 7
    loss, grad, grads = _both(x, w, labels.to(kind), "none", gen)
    values, bounds = oracle.loss_and_gradients(x.detach(), w.detach(), labels, -100, "none", grad.double().to(device))
    for name, got, want, bound in zip(("loss", "dx", "dW"), (loss, *grads), values, bounds):
        _near(got, want.cpu(), bound.cpu(), name)
    mean = linear_cross_entropy(x, w, labels.to(kind))
    count = max(1, int((labels >= 0).sum()))
    assert abs(mean.item() - values[0].sum().item() / count) <= (bounds[0].sum().item() + 2.0**-24 * 40 * values[0].sum().item()) / count


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n", [60, 300])
def test_other_gradients_through_one_graph(n, dtype, device):
    """What the forward keeps is not changed by a backward: one with other gradients gives what a graph of its own does."""
    x, w, labels, gen = _inputs(n, 300, 64, dtype, device)
    ways = [size * torch.randn(n, generator=gen).to(device) for size in (1.0, 2.0**8, 2.0**-8)]
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    for grad in ways:
        one = torch.autograd.grad(loss, (x, w), grad, retain_graph=True)
        own = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="none"), (x, w), grad)
        assert all(torch.equal(a, b) for a, b in zip(one, own))
