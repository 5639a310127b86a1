"""The example decoder: window attention and memory trained together, prompts through a cache, tokens decoded from it."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "window_decoder.py"
    spec = importlib.util.spec_from_file_location("window_decoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_training_step_reaches_every_parameter(example, device):
    torch.manual_seed(1)
    model = example.Decoder().to(device, torch.bfloat16)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    losses = example.train(model, 3, torch.Generator().manual_seed(1))
    assert all(torch.isfinite(torch.tensor(losses)))
    assert all(not torch.equal(before[n], p) for n, p in model.named_parameters() if p.grad is not None and p.grad.any())
    for name in ("attention.qkv.weight", "attention.out.weight", "embed.weight"):
        assert dict(model.named_parameters())[name].grad.abs().sum() > 0


def test_decoding_from_the_cache_follows_the_whole_forward(example, device):
    """Logits of a decode step against the forward over all tokens: the cache's 4 bits are what differs."""
    torch.manual_seed(2)
    model = example.Decoder().to(device, torch.bfloat16)
    B, T = 3, 70
    tokens = torch.randint(0, 64, (B, T), device=device)
    positions = torch.arange(T, device=device).expand(B, -1)
    with torch.no_grad():
        x = model.norm1(model.inputs(tokens, positions))
        want, k, v = model.attention(x)
        cache = example.Int4KVCache(B * 5, 2, 64, page_size=16, device=device)
        table = torch.arange(B * 5, dtype=torch.int32, device=device).view(B, 5)
        count = torch.full((B,), T - 2, dtype=torch.int32, device=device)
        cache.append(k[:, :, : T - 2], v[:, :, : T - 2], table, torch.zeros_like(count), count)
        got = model.attention.decode(x[:, T - 2 :], cache, table, count + 2)
    torch.cuda.synchronize()
    # 4 bits: numbers are off by a quarter of a step in the mean square root, a step is a fifteenth of a group's range
    # of about 4 deviations: below a tenth of the numbers; the average over the window's tokens less
    off = (got.float() - want[:, T - 2 :].float()).norm() / want[:, T - 2 :].float().norm()
    assert off < 0.2


def test_generate_takes_padded_prompts(example, device):
    """A left-padded prompt decodes to the tokens of the same prompt alone."""
    torch.manual_seed(3)
    model = example.Decoder().to(device, torch.bfloat16)
    text = torch.randint(0, 64, (1, 40), device=device)
    padded = torch.cat([torch.zeros((1, 13), dtype=torch.long, device=device), text], 1)
    zero, pad = (torch.tensor([n], dtype=torch.int32, device=device) for n in (0, 13))
    a = example.generate(model, text, zero, 6)
    b = example.generate(model, padded, pad, 6)
    assert a.shape == (1, 6)
    assert (a == b).float().mean() >= 0.5  # other tiles, other order of sums: a near tie may fall the other way
