"""Token embedding: arguments that are refused, on the CPU before any kernel runs."""
from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from modelos_amd import token_embedding as te

P = ctypes.c_void_p(1 << 20)
IDS = torch.zeros(3, dtype=torch.long)


@pytest.fixture(scope="module")
def lib():
    from modelos_amd import _lib, build_lib

    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    return _lib.load()


@pytest.mark.parametrize("ids,w,options,error", [
    (IDS, torch.zeros(4), {}, ValueError),
    (IDS, torch.zeros(4, 0), {}, ValueError),
    (IDS.short(), torch.zeros(4, 8), {}, TypeError),
    (IDS.float(), torch.zeros(4, 8), {}, TypeError),
    (IDS, torch.zeros(4, 8), {"scale": float("nan")}, ValueError),
    (IDS, torch.zeros(4, 8), {"scale": float("inf")}, ValueError),
    (IDS, torch.zeros(4, 8), {"padding_idx": 4}, ValueError),
    (IDS, torch.zeros(4, 8), {"padding_idx": -5}, ValueError),
    (IDS, torch.zeros(4, 8), {"padding_idx": True}, ValueError),
    (IDS, torch.zeros(0, 8), {"padding_idx": 0}, ValueError),
    (IDS, torch.zeros(4, 8, dtype=torch.float64), {}, NotImplementedError),
    (IDS, torch.zeros(4, 8), {}, RuntimeError),  # CPU tensors
])
def test_refused(ids, w, options, error):
    with pytest.raises(error):
        te.token_embedding(ids, w, **options)


def test_dual_tensors_are_refused():
    with forward_ad.dual_level():
        w = forward_ad.make_dual(torch.zeros(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward"):
            te.token_embedding(IDS, w)


def test_too_many():
    w = torch.zeros(1, 8).expand(1 << 31, 8)
    with pytest.raises(NotImplementedError, match="not supported"):
        te.token_embedding(IDS, w)


def test_module():
    e = te.TokenEmbedding(5, 8, padding_idx=2, scale=3.0)
    assert e.weight.shape == (5, 8) and not e.weight[2].any() and e.weight[1].any()
    assert "padding_idx=2" in repr(e)
    assert set(e.state_dict()) == {"weight"}


@pytest.mark.parametrize("args,status", [
    ((P, 16, 3, P, 4, 8, 8, 0, 1.0, P, None), 1),  # ids of 16 bits
    ((P, 64, 3, P, 4, 8, 8, 7, 1.0, P, None), 1),  # no such type
    ((P, 64, -1, P, 4, 8, 8, 0, 1.0, P, None), 1),
    ((P, 64, 3, None, 4, 8, 8, 0, 1.0, P, None), 1),
    ((None, 64, 3, P, 4, 8, 8, 0, 1.0, P, None), 1),
    ((P, 64, 3, P, 4, -1, 8, 0, 1.0, P, None), 1),
    ((P, 64, 1 << 31, P, 4, 8, 8, 0, 1.0, P, None), 2),
    ((P, 64, 3, P, 4, 8, 1 << 24, 0, 1.0, P, None), 2),
    ((P, 64, 0, None, 4, 8, 8, 0, 1.0, None, None), 0),  # nothing to do
    ((P, 64, 3, P, 4, 8, 0, 0, 1.0, P, None), 0),
])
def test_entry_forward(lib, args, status):
    assert lib.pkm_embed_fwd(*args) == status


@pytest.mark.parametrize("args,status", [
    ((P, 64, 3, P, 4, 8, 0, -1, 1.0, P, P, 0, None), 3),  # no workspace
    ((P, 64, 3, P, 4, 8, 0, -1, 1.0, None, P, 1 << 20, None), 1),
    ((P, 64, 3, None, 4, 8, 0, -1, 1.0, P, P, 1 << 20, None), 1),
    ((P, 64, 3, P, 4, 8, 0, -1, 1.0, P, ctypes.c_void_p((1 << 20) + 8), 1 << 20, None), 1),
    ((P, 64, 1 << 30, P, 4, 4096, 0, -1, 1.0, P, P, 1 << 62, None), 2),  # pieces of a launch
    ((P, 64, 3, P, 0, 8, 0, -1, 1.0, None, None, 0, None), 0),
])
def test_entry_backward(lib, args, status):
    assert lib.pkm_embed_bwd(*args) == status


def test_workspace_size(lib):
    assert lib.pkm_embed_bwd_workspace_size(0, 10, 8) == 256
    assert lib.pkm_embed_bwd_workspace_size(100, 10, 8) == 256 + 1792 + 2 * 7 * 32
    assert lib.pkm_embed_bwd_workspace_size(-1, 10, 8) == 0
