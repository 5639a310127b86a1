"""The example decoder by its values: what attention gives at each decode step of a padded prompt against the same prompt
alone, with controls that have to be seen; every parameter's gradient; the trained example's own answer.

Tokens are forced, so both runs' steps see the same inputs. Their attention may differ by the roundings of two bf16
results and of the keys and values behind them (each 2^-9 in the mean, and now and then one step of a code, 2^-7 over
all): below 2^-5 of its norm. The controls differ by whole tokens of a window of 32."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

SAME, OTHER = 2.0**-5, 2.0**-3
PAD, TEXT, NEW = 13, 40, 9


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "window_decoder.py"
    spec = importlib.util.spec_from_file_location("window_decoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def model(example):
    torch.manual_seed(3)
    return example.Decoder().to("cuda", torch.bfloat16)


def _answers(example, model, prompts, starts, forced, spoil=None):
    """What attention gives at the prompt's last token and at every step of generate(), whose tokens are `forced`."""
    found, attention = [], model.attention
    forward, decode, step, seen = attention.forward, attention.decode, model.decode, []

    def recorded_forward(*args):
        y, k, v = forward(*args)
        found.append(y[:, -1:])
        return y, k, v

    def recorded_decode(x, cache, table, lengths):
        if spoil is not None:
            spoil(cache, len(found))
        found.append(decode(x, cache, table, lengths))
        return found[-1]

    def forced_step(token, *args):
        seen.append(token)
        step(forced[:, len(seen) - 1 : len(seen)], *args)
        return torch.nn.functional.one_hot(forced[:, len(seen) : len(seen) + 1], 64).float()

    attention.forward, attention.decode, model.decode = recorded_forward, recorded_decode, forced_step
    try:
        start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        out = example.generate(model, prompts, start, forced.shape[1] - 1)
    finally:
        del attention.forward, attention.decode, model.decode
    torch.cuda.synchronize()
    assert torch.equal(out[:, 1:], forced[:, 1:-1])  # all but the prompt's own answer
    return torch.cat(found, 1).float()


def _text(example, n):
    return torch.randint(0, 64, (1, n), generator=torch.Generator().manual_seed(5)).cuda()


def _off(a, b):
    """Of each step."""
    return ((a - b).norm(dim=-1) / b.norm(dim=-1))[0]


@pytest.fixture(scope="module")
def runs(example, model, device):
    text, forced = _text(example, TEXT), _text(example, NEW + 1)
    padded = torch.cat([torch.full((1, PAD), 7, device=device), text], 1)
    return text, padded, forced, _answers(example, model, text, [0], forced)


def test_padding_changes_nothing(example, model, runs):
    text, padded, forced, alone = runs
    off = _off(_answers(example, model, padded, [PAD], forced), alone)
    assert off.shape == (NEW + 1,) and (off <= SAME).all(), off.tolist()


def test_wrong_padding_is_seen(example, model, runs):
    _, padded, forced, alone = runs
    for start in (0, PAD + 5):
        off = _off(_answers(example, model, padded, [start], forced), alone)
        assert (off >= OTHER).any(), (start, off.tolist())


def test_an_overwritten_page_is_seen(example, model, runs):
    """One page of the cache taken from another place, in the window or with the sinks."""
    text, _, forced, alone = runs
    for page in (0, 2):
        def spoil(cache, step, page=page):
            if step == 1:
                cache.codes[:, page] = cache.codes[:, 1].clone()
                cache.params[:, page] = cache.params[:, 1].clone()
        off = _off(_answers(example, model, text, [0], forced, spoil), alone)
        assert off[0] == 0 and (off[1:] >= OTHER / 2).any(), (page, off.tolist())


def test_every_parameter_has_a_gradient(example, device):
    torch.manual_seed(1)
    model = example.Decoder().to(device, torch.bfloat16)
    example.train(model, 1, torch.Generator().manual_seed(1))
    without = [n for n, p in model.named_parameters() if p.grad is None or not p.grad.any()]
    assert without == []
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


def test_the_trained_example_goes_on(example, device):
    """Every token has one successor, which a trained layer knows: nearly all decoded tokens are right (by chance, 1 of 64)."""
    result = example.main(["--steps", "300", "--tokens", "12"])
    assert result["losses"][-1] < 0.2 * result["losses"][0]
    assert result["right"] >= 0.9
