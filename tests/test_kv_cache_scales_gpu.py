"""Attention over the 4-bit cache where steps differ between groups and tokens, and how close it is for ordinary ones.

Element by element, the kernel's roundings (u = eps / 2 of the cache's type):
- weights times steps enter as f16 numbers, off by 2^-11 of their value (f16 caches: two numbers, 2^-22) or by 2^-25 where
  that is more, in units in which the row's largest weight times its group's largest step is at least a quarter (15 of those
  units a token, for its code);
- weights times minima as two numbers of the cache's type: u^2, f16 caches with 2^-25 below the normal numbers;
- the result: u. Logits, exponentials and sums: float32.
Group by group, 2-norm of the error over that of a correctly rounded result: below 1.25, as the weights' roundings are an
eighth of a bf16 result's, independent from token to token, on numbers up to four times the result's."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.kv_cache import Int4KVCache
from oracle import attention as attn
from oracle import kv_cache as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64)]
TYPE_IDS = ["bf16-128", "bf16-64", "f16-128", "f16-64"]


def _int(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _cache(device, k, v, P, lengths, g):
    """k, v [B, H, T, D] in a cache, its table."""
    B, H, T, D = k.shape
    width = -(-T // P)
    table = torch.randperm(B * width + 2, generator=g)[: B * width].view(B, width).to(torch.int32)
    cache = Int4KVCache(B * width + 2, H, D, page_size=P, dtype=k.dtype, device=device)
    cache.params.fill_(float("nan"))
    cache.append(k.to(device), v.to(device), table.to(device), _int([0] * B, device), _int(lengths, device))
    return cache, table


def _check(device, k, v, q, P, lengths, window=None, sinks=0, limit=1.25, seed=0):
    dtype, D, Q = q.dtype, q.shape[3], q.shape[2]
    cache, table = _cache(device, k, v, P, lengths, gen(seed))
    got = cache.attend(q.to(device), table.to(device), _int(lengths, device), window=window, sinks=sinks).cpu()
    codes, params = cache.codes.cpu(), cache.params.cpu()
    f16 = dtype == torch.float16
    u = torch.finfo(dtype).eps / 2
    off, rounded = (torch.zeros(D // 32, dtype=torch.float64) for _ in range(2))
    tiny = torch.finfo(dtype).smallest_normal * u
    for b, n in enumerate(lengths):
        kk, vv = (ref.sequence(codes, params, table[b].tolist(), n, side) for side in range(2))
        km, vm = (ref.sequence(torch.zeros_like(codes), params, table[b].tolist(), n, side) for side in range(2))
        G = q.shape[1] // kk.shape[0]
        kk, vv, km, vm = (x.repeat_interleave(G, 0) for x in (kk, vv, km, vm))
        p, j = n - Q + torch.arange(Q)[:, None], torch.arange(n)[None]
        mask = (j <= p) & ((p - j < (window or n + 1)) | (j < sinks))
        x, scale = q[b].double(), D**-0.5
        s = torch.where(mask, x @ kk.transpose(1, 2) * scale, -torch.inf)
        es = 2.0**-24 * ((D + 16) * scale * (x.abs() @ ((kk - km).abs() + km.abs()).transpose(1, 2)) + 4 * s.abs() + 16)
        e = torch.where(mask, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
        w = e / e.sum(-1, keepdim=True)
        ew = w * (2 * torch.where(mask, es, 0.0).amax(-1, keepdim=True) + 2.0**-20)
        sc, mm = (vv - vm).abs(), vm.abs()
        out = w @ vv
        # each group's largest step among the tokens that any row sees
        step = torch.where(mask.any(0)[:, None], sc, 0.0).unflatten(-1, (-1, 32)).amax((1, 3))  # 1 to 15 steps
        step = step.repeat_interleave(32, -1)[:, None]
        unit = w.amax(-1, keepdim=True) * step * 2.0**-25 * 4 * 15 * mask.sum(-1, keepdim=True)
        low = (u * u * w + torch.where(mask, 2.0**-25 * w.amax(-1, keepdim=True) if f16 else 0.0, 0.0)) @ mm
        bound = (w * (2.0**-22 if f16 else 2.0**-11)) @ sc + unit + low + ew @ (sc + mm) + u * out.abs() + tiny + 1e-300
        attn.assert_within(got[b], out, bound + 2.0**-20 * (w @ (sc + mm)), f"sequence {b}")
        size = lambda x: x.square().unflatten(-1, (-1, 32)).sum((0, 1, 3))
        off += size(got[b].double() - out)
        rounded += size(out.to(dtype).double() - out)
    ratio = (off / rounded).sqrt()
    assert (ratio <= limit).all(), f"groups' errors over those of a rounded result: {ratio.tolist()}"


def _x(g, B, H, T, D, dtype):
    return torch.randn((B, T, H, D), generator=g).transpose(1, 2)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("Hq,H,Q,P,lengths,window,sinks", [
    (8, 2, 1, 64, [700, 513, 90], None, 0), (14, 2, 5, 16, [300, 77], 100, 3), (4, 4, 1, 32, [64, 65, 100], None, 0),
    (2, 2, 1, 64, [3000], 1000, 4), (2, 1, 17, 16, [130], None, 0),
])
def test_ordinary_numbers(device, dtype, D, Hq, H, Q, P, lengths, window, sinks):
    g = gen(sum(lengths))
    B, T = len(lengths), max(lengths)
    k, v, q = (_x(g, B, h, n, D, dtype) for h, n in ((H, T), (H, T), (Hq, Q)))
    k = k + torch.randn((1, H, 1, D), generator=g) / 2
    _check(device, k.to(dtype), v.to(dtype), q.to(dtype), P, lengths, window, sinks)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("ratio", [6, 12])
@pytest.mark.parametrize("form", ["groups", "tokens", "late", "early", "flat-groups", "offset"])
def test_steps_of_different_sizes(device, dtype, D, ratio, form):
    g = gen(ratio)
    B, H, T, P = 2, 2, 700, 32
    lengths = [700, 333]
    k, v, q = _x(g, B, H, T, D, dtype), _x(g, B, H, T, D, dtype), _x(g, B, 4, 1, D, dtype)
    small = 2.0**-ratio
    if form == "groups":  # channels of a head far larger than the others
        v[..., 32:] *= small
        k[..., 32:] *= small
    elif form == "tokens":
        v = v * torch.exp2(-ratio * torch.rand((B, H, T, 1), generator=g))
    elif form == "late":  # the largest step comes last
        v[:, :, :300] *= small
        v[0, :, 300:650] *= small
    elif form == "early":
        v[:, :, 33:] *= small
    elif form == "flat-groups":  # no spread beside wide groups, and in whole tokens
        v[..., :32] = v[..., :1]
        v[:, :, 100:200] = 0.0
        v[:, :, 200:300] = 2.0**ratio
    else:  # a common part much larger than the steps
        v = v * small + torch.randn((1, H, 1, D), generator=g)
    _check(device, k.to(dtype), v.to(dtype), q.to(dtype), P, lengths)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("size", [0.0, 1.0, 2.0**-20, 2.0**13, 2.0**40, 2.0**100])
def test_values_without_any_step(device, dtype, D, size):
    """Groups of equal numbers only: nothing but minima, of any size."""
    if dtype == torch.float16 and size > 2.0**13:
        pytest.skip("past float16")
    g = gen(4)
    B, H, T, P = 2, 2, 150, 16
    k, q = _x(g, B, H, T, D, dtype), _x(g, B, 4, 1, D, dtype)
    v = torch.randn((B, H, T, D // 32, 1), generator=g).expand(B, H, T, D // 32, 32).flatten(3) * size
    k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
    if size == 0.0:
        cache, table = _cache(device, k, v, P, [T, 33], g)
        assert (cache.attend(q.to(device), table.to(device), _int([T, 33], device)) == 0).all()
        return
    _check(device, k, v, q, P, [T, 33])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [2.0**-90, 2.0**-40, 2.0**40, 2.0**90])
def test_steps_of_any_size(device, D, size):
    g = gen(6)
    B, H, T, P = 1, 2, 300, 64
    k, v, q = _x(g, B, H, T, D, None), _x(g, B, H, T, D, None) * size, _x(g, B, 2, 1, D, None)
    bf16 = torch.bfloat16
    k, v, q = k.to(bf16), v.to(bf16), q.to(bf16)
    cache, table = _cache(device, k, v, P, [T], gen(0))
    unit, _ = _cache(device, k, (v.double() / size).to(bf16), P, [T], gen(0))
    a, b = (c.attend(q.to(device), table.to(device), _int([T], device)) for c in (cache, unit))
    assert torch.equal(a.double() / size, b.double())
