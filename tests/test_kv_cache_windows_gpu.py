"""Attention over the cache through windows and sinks longer than 2^24 tokens: a long sequence whose positions share
two pages, one of zeros and one whose keys outweigh all the others."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.kv_cache import Int4KVCache

pytestmark = pytest.mark.gpu

P, N = 4096, 25_000_000


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("window,sinks,at,seen", [
    (20_000_000, 0, 6_000_000, True), (20_000_000, 0, 4_900_000, False), (16_000_000, 0, 6_000_000, False),
    (None, 0, 100_000, True), (10, 17_500_000, 17_200_000, True), (10, 17_500_000, 17_600_000, False),
])
def test_keys_far_behind(device, dtype, window, sinks, at, seen):
    cache = Int4KVCache(2, 1, 64, page_size=P, dtype=dtype, device=device)
    x = torch.full((1, 1, P, 64), 4.0, dtype=dtype, device=device)
    one = lambda *n: torch.tensor(n, dtype=torch.int32, device=device)
    cache.append(x, x * 0.75, one(1)[:, None], one(0), one(P))
    table = torch.zeros((1, -(-N // P)), dtype=torch.int32, device=device)
    table[0, at // P] = 1  # logits of 128 and values of 3; 0 elsewhere
    out = cache.attend(x[:, :, :1], table, one(N), window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert (out == (3.0 if seen else 0.0)).all()
