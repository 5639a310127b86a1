"""Windows and sinks of attention over the cache are taken as they are given, up to the longest sequence a cache may hold.
CPU only: what the entry point is handed."""
from __future__ import annotations

import pytest
import torch

from modelos_amd import kv_cache

I32 = torch.int32
MOST = 1 << 30  # positions of a sequence that the entry point takes are below


@pytest.fixture
def handed(monkeypatch):
    calls = []
    monkeypatch.setattr(kv_cache, "_require_device", lambda *tensors: None)
    monkeypatch.setattr(kv_cache._lib, "call_on", lambda device, name, *args: calls.append((name, args)))
    monkeypatch.setattr(kv_cache._lib, "stream_of", lambda device: 0)
    return calls


@pytest.mark.parametrize("window,sinks", [(None, 0), (7, 3), (1 << 24, 1 << 24), (20_000_000, 18_000_000), (MOST - 1, MOST - 1),
                                          (MOST, MOST), (1 << 70, 1 << 70)])
def test_windows_are_not_cut(handed, window, sinks):
    cache = kv_cache.Int4KVCache(2, 2, 64, page_size=16, device="cpu")
    q = torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16)
    cache.attend(q, torch.zeros((1, 2), dtype=I32), torch.full((1,), 5, dtype=I32), window=window, sinks=sinks)
    (name, args), = handed
    assert name == "pkm_kv4_attend"
    # codes, params, pages, heads, page, dim, dtype, q, table, width, lengths, batch, q_heads, queries, window, sinks
    got_window, got_sinks = args[14], args[15]
    see = lambda gap, w: w == 0 or gap < w
    for gap in (0, 6, 7, (1 << 24) - 1, 1 << 24, 17_000_000, 20_000_000, MOST - 2, MOST - 1):
        assert see(gap, got_window) == see(gap, window or 0), gap
        assert (gap < got_sinks) == (gap < sinks), gap
    assert max(got_window, got_sinks) < 1 << 63
