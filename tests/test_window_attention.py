"""Refusals of window attention, before any kernel runs. CPU only."""
from __future__ import annotations

import ctypes

import pytest
import torch

from modelos_amd.window_attention import window_attention


def _heads(H=4, T=8, D=64, B=2, dtype=torch.bfloat16):
    return torch.zeros((B, H, T, D), dtype=dtype)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=2.0), dict(window=True), dict(sinks=-1),
                                dict(sinks=1.5), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(starts=torch.zeros(2)),
                                dict(ends=torch.zeros(3, dtype=torch.int32))])
def test_bad_options(kw):
    with pytest.raises(ValueError):
        window_attention(_heads(), _heads(2), _heads(2), **kw)


@pytest.mark.parametrize("q,k,v", [
    (_heads(), _heads(3), _heads(3)), (_heads(), _heads(2), _heads(4)), (_heads(), _heads(2, T=9), _heads(2, T=9)),
    (_heads(), _heads(2, B=1), _heads(2, B=1)), (_heads(), _heads(2, D=128), _heads(2, D=128)),
    (_heads()[0], _heads(2)[0], _heads(2)[0]), (_heads(), _heads(0), _heads(0)),
])
def test_bad_shapes(q, k, v):
    with pytest.raises(ValueError):
        window_attention(q, k, v)


@pytest.mark.parametrize("t", [_heads(2, dtype=torch.float32), _heads(2, D=80), _heads(2, D=256)])
def test_unsupported(t):
    with pytest.raises(NotImplementedError):
        window_attention(t, t, t)


def test_mixed_types_and_cpu_tensors():
    with pytest.raises(NotImplementedError):
        window_attention(_heads(), _heads(2, dtype=torch.float16), _heads(2, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        window_attention(_heads(), _heads(2), _heads(2))


@pytest.fixture(scope="module")
def lib():
    from modelos_amd import _lib, build_lib

    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    return _lib.load()


def _fwd(lib, x, sizes=(1, 4, 2, 8, 64, 1), window=0, sinks=0, scale=0.1):
    return lib.pkm_window_attn_fwd(x, x, x, None, None, *sizes, window, sinks, scale, x, None, None, None)


def test_entry_point_statuses(lib):
    from modelos_amd._lib import Heads

    good = Heads(1 << 20, 2048, 512, 64)
    assert _fwd(lib, None) == 1
    assert b"q is NULL" in lib.pkm_last_error_string()
    assert _fwd(lib, Heads(None, 2048, 512, 64)) == 1
    assert _fwd(lib, good, (1, 4, 3, 8, 64, 1)) == 1
    assert _fwd(lib, good, (1, 4, 2, -1, 64, 1)) == 1
    assert _fwd(lib, good, (1, 4, 0, 8, 64, 1)) == 1
    assert _fwd(lib, good, window=-1) == 1
    assert _fwd(lib, good, sinks=-1) == 1
    assert _fwd(lib, good, scale=0.0) == 1
    assert _fwd(lib, good, scale=float("nan")) == 1
    assert _fwd(lib, good, (1, 4, 2, 8, 96, 1)) == 2
    assert _fwd(lib, good, (1, 4, 2, 8, 64, 0)) == 2
    assert _fwd(lib, good, (1, 4, 2, 1 << 24, 64, 1)) == 2
    assert _fwd(lib, good, (1 << 40, 1 << 40, 1, 8, 64, 1)) == 2
    assert _fwd(lib, Heads((1 << 20) + 8, 2048, 512, 64)) == 2
    assert _fwd(lib, Heads(1 << 20, 2048, 512, 68)) == 2
    assert _fwd(lib, Heads(1 << 20, 2048, 512, 1 << 22)) == 2
    assert _fwd(lib, Heads(1 << 20, 2048, 512, -64)) == 2
    # nothing to do: no kernel
    assert _fwd(lib, None, (0, 4, 2, 8, 64, 1)) == 0
    assert _fwd(lib, None, (1, 4, 2, 0, 64, 1)) == 0


def test_backward_workspace(lib):
    from modelos_amd._lib import Heads

    x = Heads(1 << 20, 2048, 512, 64)
    sizes = (1, 4, 2, 8, 64)
    need = lib.pkm_window_attn_bwd_workspace_size(*sizes, 0, 0)
    assert need >= 4 * 8 * 4
    assert lib.pkm_window_attn_bwd_workspace_size(-1, 4, 2, 8, 64, 0, 0) == 0
    lse = ctypes.c_void_p(1 << 20)
    run = lambda lse, ws, n: lib.pkm_window_attn_bwd(x, x, x, x, None, lse, x, None, None, *sizes, 1, 0, 0, 0.1, x, x, x, ws,
                                                     n, None)
    assert run(None, lse, need) == 1
    assert run(lse, None, need) == 3
    assert run(lse, lse, need - 1) == 3
