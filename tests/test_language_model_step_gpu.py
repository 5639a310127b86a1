"""Tokens in, loss out, update: embedding, loss and AdamW together, as a training step runs them."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F
import torch.utils.checkpoint

from modelos_amd.adamw import AdamW
from modelos_amd.linear_cross_entropy import linear_cross_entropy
from modelos_amd.token_embedding import token_embedding

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
VOCAB, DIM, TOKENS = 700, 72, 500


def _weights(device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    table = 0.2 * torch.randn((VOCAB, DIM), generator=gen)
    gate = 1 + 0.3 * torch.randn(DIM, generator=gen)
    return [x.to(BF16).to(device).requires_grad_() for x in (table, gate)]


def _batch(device, seed):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, (TOKENS + 1,), generator=gen)
    labels = torch.where(torch.rand(TOKENS, generator=gen) < 0.2, -100, ids[1:])
    return ids[:-1].to(device), labels.to(device)


def _loss(table, gate, ids, labels):
    """A model without a library's products: embedded tokens, gated and shifted by one, against the same table."""
    x = token_embedding(ids, table, scale=2.0, padding_idx=3)
    return linear_cross_entropy(x * gate + x.roll(1, 0), table, labels)


def test_gradients_of_a_tied_table(device):
    """Both ends' gradients meet in the table. Against autograd in 64 bits of the same formulas: eight roundings to bf16 lie
    between (out, product, sum, the logits' gradients, dhidden, product, both gradients and their sum), each 2^-8 of what it
    rounds at most; the two ends' gradients do not cancel."""
    table, gate = _weights(device)
    ids, labels = _batch(device, 1)
    got = torch.autograd.grad(_loss(table, gate, ids, labels), (table, gate))
    t, g = (x.detach().cpu().double().requires_grad_() for x in (table, gate))
    read = torch.where((ids.cpu() == 3)[:, None], t.detach()[ids.cpu()], t[ids.cpu()]) * 2
    want = torch.autograd.grad(F.cross_entropy((read * g + read.roll(1, 0)) @ t.T, labels.cpu()), (t, g))
    for a, b in zip(got, want):
        assert (a.cpu().double() - b).norm() <= 8 * 2**-8 * b.norm()


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_are_the_eager_ones(bits, device):
    """Five steps of a graph and five eager ones leave the same bits: batches change, the step counts on."""
    ids, labels = (torch.zeros(TOKENS, dtype=torch.long, device=device) for _ in range(2))

    def model():
        weights = _weights(device)
        return weights, AdamW(weights, lr=1e-2, betas=(0.9, 0.95), state_bits=bits, master_weights=True)

    def step(weights, opt):
        loss = _loss(*weights, ids, labels)
        for p, g in zip(weights, torch.autograd.grad(loss, weights)):
            p.grad = g
        opt.step()
        return loss.detach()

    batch = lambda k: [x.copy_(y) for x, y in zip((ids, labels), _batch(device, k))]
    eager, captured = model(), model()
    batch(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*captured)  # the first one, which makes the states
    torch.cuda.current_stream().wait_stream(side)
    first = step(*eager)
    assert all(torch.equal(a, b) for a, b in zip(eager[0], captured[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(*captured)
    losses = [first.item()]
    for k in range(1, 6):
        batch(k)
        graph.replay()
        want = step(*eager)
        assert torch.equal(loss, want)
        assert all(torch.equal(a, b) for a, b in zip(eager[0], captured[0]))
        for a, b in zip(eager[0], captured[0]):
            assert all(torch.equal(x.float(), captured[1].state[b][n].float()) for n, x in eager[1].state[a].items())
        losses.append(want.item())
    assert all(x == x and x < 20 for x in losses)


def test_two_streams_at_once(device):
    """Two models' steps on two streams, side by side, leave what each leaves alone."""
    def run(seed, stream):
        weights = _weights(device, seed)
        opt = AdamW(weights, lr=1e-2)
        ids, labels = _batch(device, seed)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(3):
                for p, g in zip(weights, torch.autograd.grad(_loss(*weights, ids, labels), weights)):
                    p.grad = g
                opt.step()
                yield
        yield weights

    alone = []
    for seed in (4, 5):
        *_, weights = run(seed, torch.cuda.current_stream())
        alone.append(weights)
    torch.cuda.synchronize()
    both = [run(seed, torch.cuda.Stream()) for seed in (4, 5)]
    for _ in range(3):
        for r in both:
            next(r)
    got = [next(r) for r in both]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(alone, got) for a, b in zip(x, y))


def test_the_example_decoder_trains_through_them(device):
    """Its loss and every gradient against F.cross_entropy of its logits, which bf16 rounds: logits up to 2 are off by 2^-8,
    softmax weights by as much of themselves, gradients by a few times 2^-8 in the norm."""
    path = Path(__file__).resolve().parents[1] / "examples" / "window_decoder.py"
    spec = importlib.util.spec_from_file_location("window_decoder", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(1)
    model = example.Decoder().to(device, BF16)
    tokens = torch.randint(0, 64, (4, 65), device=device)
    positions = torch.arange(64, device=device).expand(4, -1)
    params = list(model.parameters())
    loss = model.loss(tokens[:, :-1], positions, tokens[:, 1:])
    got = torch.autograd.grad(loss, params)
    logits, _, _ = model(tokens[:, :-1], positions)
    want_loss = F.cross_entropy(logits.flatten(0, 1).float(), tokens[:, 1:].flatten())
    want = torch.autograd.grad(want_loss, params)
    assert abs(loss.item() - want_loss.item()) <= 2**-8 * 4
    for (name, _), a, b in zip(model.named_parameters(), got, want):
        assert (a.float() - b.float()).norm() <= 8 * 2**-8 * b.float().norm(), name


@pytest.mark.parametrize("tokens", [40, 500])
def test_gradients_twice_and_recomputed(tokens, device):
    """The same bits from one graph twice, and where a checkpoint runs the forward again."""
    table, gate = _weights(device)
    ids, labels = (x[:tokens] for x in _batch(device, 2))
    loss = _loss(table, gate, ids, labels)
    first = torch.autograd.grad(loss, (table, gate), retain_graph=True)
    again = torch.autograd.grad(loss, (table, gate))
    loss = torch.utils.checkpoint.checkpoint(_loss, table, gate, ids, labels, use_reentrant=False)
    for a, b, c in zip(first, again, torch.autograd.grad(loss, (table, gate))):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_labels_and_ids_of_one_value(device):
    """All tokens the same id, all labels the same entry: every sum of the step is one row's."""
    table, gate = _weights(device)
    ids, labels = torch.full((TOKENS,), 5, device=device), torch.full((TOKENS,), 5, device=device)
    got = torch.autograd.grad(_loss(table, gate, ids, labels), (table, gate))
    t, g = (x.detach().cpu().double().requires_grad_() for x in (table, gate))
    read = t[ids.cpu()] * 2
    want = torch.autograd.grad(F.cross_entropy((read * g + read.roll(1, 0)) @ t.T, labels.cpu()), (t, g))
    for a, b in zip(got, want):  # the roundings of test_gradients_of_a_tied_table; those of equal tokens add up as the values do
        assert (a.cpu().double() - b).norm() <= 8 * 2**-8 * b.norm()
