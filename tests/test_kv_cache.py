"""The 4-bit cache's refusals before any kernel runs, and the oracle's own consistency. CPU only."""
from __future__ import annotations

import ctypes

import pytest
import torch

from modelos_amd.kv_cache import Int4KVCache
from oracle import kv_cache as ref

I32 = torch.int32


@pytest.mark.parametrize("D", [64, 128])
def test_oracle_codes_come_back(D):
    c = torch.randint(0, 16, (3, 5, D))
    assert torch.equal(ref.unpack(ref.pack(c), D), c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_oracle_numbers_lie_within_half_a_step(dtype):
    x = torch.randn((50, 128)).to(dtype)
    c, s, m = ref.quantise(x)
    off = (ref.values(c, s, m) - x.double()).abs().unflatten(-1, (-1, 32)).amax(-1)
    # half a step, and 15 times the rounding of the step
    assert (off <= s.double() * (0.5 + 15 * torch.finfo(dtype).eps / 2 * 1.01)).all()


@pytest.mark.parametrize("kw,error", [
    (dict(pages=0), ValueError), (dict(kv_heads=0), ValueError), (dict(page_size=0), ValueError),
    (dict(pages=1.5), ValueError), (dict(dim=96), NotImplementedError), (dict(dtype=torch.float32), NotImplementedError),
    (dict(page_size=24), NotImplementedError), (dict(page_size=8192), NotImplementedError),
])
def test_bad_caches(kw, error):
    args = dict(pages=2, kv_heads=2, dim=64, page_size=16, dtype=torch.bfloat16)
    args.update(kw)
    with pytest.raises(error):
        Int4KVCache(args["pages"], args["kv_heads"], args["dim"], page_size=args["page_size"], dtype=args["dtype"],
                    device="cpu")


def _cache():
    return Int4KVCache(4, 2, 64, page_size=16, device="cpu")


def _x(H=2, T=3, D=64, B=2, dtype=torch.bfloat16):
    return torch.zeros((B, H, T, D), dtype=dtype)


TABLE, N = torch.zeros((2, 2), dtype=I32), torch.ones(2, dtype=I32)


@pytest.mark.parametrize("k,v,table,starts,counts", [
    (_x(3), _x(3), TABLE, N, N), (_x(), _x(T=4), TABLE, N, N), (_x(D=128), _x(D=128), TABLE, N, N),
    (_x(dtype=torch.float16), _x(dtype=torch.float16), TABLE, N, N), (_x()[0], _x()[0], TABLE, N, N),
    (_x(), _x(), TABLE.long(), N, N), (_x(), _x(), TABLE[0], N, N), (_x(), _x(), TABLE[:1], N, N),
    (_x(), _x(), TABLE, N.long(), N), (_x(), _x(), TABLE, N[:1], N), (_x(), _x(), TABLE, N, N[None]),
])
def test_bad_appends(k, v, table, starts, counts):
    with pytest.raises(ValueError):
        _cache().append(k, v, table, starts, counts)


def test_bad_reads():
    with pytest.raises(ValueError):
        _cache().read(TABLE, N, N, -1)
    with pytest.raises(ValueError):
        _cache().read(TABLE, N, N[:1], 2)


@pytest.mark.parametrize("q,kw", [
    (_x(3), {}), (_x(D=128), {}), (_x(dtype=torch.float16), {}), (_x()[0], {}), (_x(4), dict(window=0)),
    (_x(4), dict(sinks=-1)), (_x(4), dict(scale=0.0)), (_x(4, B=3), {}),
])
def test_bad_attends(q, kw):
    with pytest.raises(ValueError):
        _cache().attend(q, TABLE, N, **kw)


def test_attend_has_no_backward_and_no_cpu_path():
    with pytest.raises(RuntimeError, match="no backward"):
        _cache().attend(_x(4).requires_grad_(True), TABLE, N)
    with pytest.raises(RuntimeError, match="no CPU path"):
        _cache().attend(_x(4), TABLE, N)
    with pytest.raises(RuntimeError, match="no CPU path"):
        _cache().append(_x(), _x(), TABLE, N, N)


@pytest.fixture(scope="module")
def lib():
    from modelos_amd import _lib, build_lib

    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    return _lib.load()


P = ctypes.c_void_p(1 << 20)


def _append(lib, x, sizes=(4, 2, 16, 64, 1), codes=P, counts=P, batch=2, tokens=3, table=P, width=2):
    return lib.pkm_kv4_append(codes, P, *sizes, x, x, table, width, P, counts, batch, tokens, None)


def _attend(lib, x, sizes=(4, 2, 16, 64, 1), width=2, lengths=P, heads=4, queries=1, window=0, sinks=0, scale=0.1,
            ws=None, n=0, batch=2):
    return lib.pkm_kv4_attend(P, P, *sizes, x, P, width, lengths, batch, heads, queries, window, sinks, scale, x, ws, n,
                              None)


def test_entry_point_statuses(lib):
    from modelos_amd._lib import Heads

    good = Heads(1 << 20, 2048, 512, 64)
    assert _append(lib, None) == 1
    assert _append(lib, good, codes=None) == 1
    assert _append(lib, good, counts=None) == 1
    assert _append(lib, good, table=None) == 1
    assert _append(lib, good, batch=-1) == 1
    assert _append(lib, good, (4, 0, 16, 64, 1)) == 1
    assert _append(lib, good, (4, 2, 24, 64, 1)) == 2
    assert _append(lib, good, (4, 2, 16, 96, 1)) == 2
    assert _append(lib, good, (4, 2, 16, 64, 0)) == 2
    assert _append(lib, good, tokens=1 << 31) == 2
    assert _append(lib, good, batch=(1 << 31) - 1, tokens=(1 << 31) - 1) == 2
    assert _append(lib, good, batch=1 << 62) == 2
    assert _append(lib, Heads((1 << 20) + 4, 2048, 512, 64)) == 2
    assert _append(lib, good, batch=0) == 0
    assert _append(lib, good, tokens=0) == 0
    assert _attend(lib, None) == 1
    assert _attend(lib, good, lengths=None) == 1
    assert _attend(lib, good, heads=3) == 1
    assert _attend(lib, good, window=-1) == 1
    assert _attend(lib, good, scale=-0.1) == 1
    assert _attend(lib, good, (4, 2, 16, 80, 1)) == 2
    assert _attend(lib, good, (0, 2, 16, 64, 1)) == 2
    assert _attend(lib, good, width=1 << 30) == 2
    assert _attend(lib, good, queries=1 << 24) == 2
    assert _attend(lib, good, batch=1 << 23, heads=1 << 23, queries=1 << 23) == 2
    assert lib.pkm_kv4_attend_workspace_size(1 << 23, 1 << 23, 1, 1 << 23, 64, 4, 16, 0, 0) == 0
    assert _attend(lib, Heads(1 << 20, 2044, 512, 64)) == 2
    assert _attend(lib, good, queries=0) == 0
    assert _attend(lib, good, batch=0) == 0
    need = lib.pkm_kv4_attend_workspace_size(2, 4, 2, 1, 64, 4096, 16, 0, 0)
    assert need > 0
    assert _attend(lib, good, width=4096) == 3
    assert _attend(lib, good, width=4096, ws=P, n=need - 1) == 3
    assert lib.pkm_kv4_attend_workspace_size(0, 4, 2, 1, 64, 4, 16, 0, 0) == 0
    assert lib.pkm_kv4_attend_workspace_size(2, 4, 2, 0, 64, 4, 16, 0, 0) == 0
