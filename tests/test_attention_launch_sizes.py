"""The largest calls of window attention and of the 4-bit cache: sizes that one launch does not take are refused as unsupported. CPU only."""
from __future__ import annotations

import ctypes

import pytest

P = ctypes.c_void_p(1 << 20)
UNSUPPORTED = 2


@pytest.fixture(scope="module")
def lib():
    from modelos_amd import _lib, build_lib

    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    return _lib.load()


def _store(lib, entry, heads, dim, batch, tokens):
    from modelos_amd._lib import Heads

    x = Heads(1 << 20, 0, 0, 0)
    cache = (P, P, 4, heads, 16, dim, 1)
    if entry == "append":
        return lib.pkm_kv4_append(*cache, x, x, P, 2, P, P, batch, tokens, None)
    return lib.pkm_kv4_read(*cache, P, 2, P, P, batch, tokens, x, x, None)


@pytest.mark.parametrize("entry,heads,dim,batch,tokens", [
    ("read", 8, 128, 64, 1 << 18), ("read", 1, 64, 2, 1 << 27), ("read", 16, 128, 1, 1 << 23),
    ("append", 8, 128, 64, 1 << 20), ("append", 1, 128, 1 << 9, 1 << 20),
])
def test_threads_of_one_launch(lib, entry, heads, dim, batch, tokens):
    lanes = dim // (32 if entry == "append" else 8)
    assert 2 * batch * tokens * heads * lanes >= 1 << 32
    assert _store(lib, entry, heads, dim, batch, tokens) == UNSUPPORTED
    assert b"too many tokens" in lib.pkm_last_error_string()


def test_rows_of_one_launch(lib):
    from modelos_amd._lib import Heads

    x = Heads(1 << 20, 0, 0, 0)
    run = lambda batch: lib.pkm_kv4_attend(P, P, 4, 1, 16, 64, 1, x, P, 2, P, batch, 1, 1, 0, 0, 0.1, x, None, 0, None)
    assert run((1 << 24) - 1) == UNSUPPORTED  # and 768 workgroups more
    assert run((1 << 24) - 1024) == 3  # only the workspace is missing
    size = lambda batch: lib.pkm_kv4_attend_workspace_size(batch, 1, 1, 1, 64, 2, 16, 0, 0)
    assert size((1 << 24) - 1) == 0 and size((1 << 24) - 1024) > 0


@pytest.mark.parametrize("batch,q_heads,kv_heads,tokens,status", [
    ((1 << 24) - 1, 1, 1, 1, UNSUPPORTED),  # dK and dV: 512 threads for each
    (1 << 22, 3, 3, 1, UNSUPPORTED), ((1 << 23) - 1, 1, 1, 1, 3), (1 << 20, 12, 12, 200, UNSUPPORTED),
    (1 << 10, 16, 4, 1 << 15, 3),  # 2^29 rows: large, but taken
])
def test_window_attention_of_one_launch(lib, batch, q_heads, kv_heads, tokens, status):
    from modelos_amd._lib import Heads

    x = Heads(1 << 20, 0, 0, 0)
    got = lib.pkm_window_attn_bwd(x, x, x, x, None, P, x, None, None, batch, q_heads, kv_heads, tokens, 64, 1, 0, 0, 0.1, x, x, x,
                                  None, 0, None)
    assert got == status  # 3: only the workspace is missing
