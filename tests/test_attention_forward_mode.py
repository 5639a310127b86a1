"""Attention has no forward-mode derivatives: dual tensors are refused instead of losing their tangents. CPU only, before
any kernel runs."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from modelos_amd import kv_cache, window_attention as wa

I32 = torch.int32


@pytest.fixture(autouse=True)
def no_kernels(monkeypatch):
    """Everything up to the entry points, whose outputs are zeros."""
    for module in (wa, kv_cache):
        monkeypatch.setattr(module, "_require_device", lambda *tensors: None)
        monkeypatch.setattr(module._lib, "call_on", lambda *args: None)
        monkeypatch.setattr(module._lib, "stream_of", lambda device: 0)


def _heads(H):
    return torch.randn((1, H, 5, 64)).to(torch.bfloat16)


def _window(q, k, v):
    return wa.window_attention(q, k, v, window=3)


def _attend(q, k, v):
    cache = kv_cache.Int4KVCache(2, 2, 64, page_size=16, device="cpu")
    return cache.attend(q, torch.zeros((1, 2), dtype=I32), torch.full((1,), 5, dtype=I32))


@pytest.mark.parametrize("call,dual", [(_window, 0), (_window, 1), (_window, 2), (_attend, 0)],
                         ids=["window-q", "window-k", "window-v", "cache-q"])
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(call, dual, grad):
    x = [_heads(4), _heads(2), _heads(2)]
    with torch.set_grad_enabled(grad):
        assert call(*x).shape == x[0].shape  # without tangents the call goes through
        with forward_ad.dual_level():
            assert call(*x).shape == x[0].shape
            x[dual] = forward_ad.make_dual(x[dual], torch.ones_like(x[dual]))
            with pytest.raises(NotImplementedError, match="forward"):
                call(*x)


@pytest.mark.parametrize("call", [_window, _attend])
def test_jvp_is_refused(call):
    x = [_heads(4), _heads(2), _heads(2)]
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda q: call(q, *x[1:]), (x[0],), (torch.ones_like(x[0]),))
