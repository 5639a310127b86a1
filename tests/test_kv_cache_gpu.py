"""The 4-bit key / value cache: append and read exactly, attention over it against the formulas in 64 bits.

Bounds of attend: weights with the values' steps in them may be rounded to bf16 (u = 2^-8; f16 caches: to a bf16 and
the rest in bf16, 2^-16), weights of the minima to the cache's type, codes may enter the product as 16 + c; the result
is rounded to the cache's type. The kernel rounds its weights more finely than that."""
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


def _table(B, width, pages, g):
    return torch.randperm(pages, generator=g)[: B * width].view(B, width).to(torch.int32)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("P,H,T,starts,counts", [
    (16, 3, 1, [0, 15, 16, 47], [1, 1, 1, 0]), (16, 2, 21, [0, 5, 15, 27], [21, 20, 7, 0]),
    (64, 1, 130, [0, 63, 100], [130, 129, 1]), (48, 4, 33, [10, 0], [33, 40]),
])
def test_append_and_read_exactly(device, dtype, D, P, H, T, starts, counts):
    """Codes, parameters and numbers bit for bit; nothing else changes."""
    g = gen(1)
    B = len(starts)
    width = max(-(-(s + T) // P) for s in starts)
    pages = B * width + 2
    table = _table(B, width, pages, g)
    x = torch.randn((2, B, T, H, D), generator=g) * torch.exp(torch.randn((2, B, T, H, 1), generator=g) * 2)
    x[0, 0, 0, 0, :32] = 1.25  # a group without spread
    x[1, 0, 0, 0, 32:64] = torch.arange(32) % 16  # every code, exactly
    x[1, 0, 0, 0, :32] = torch.arange(32) / 2  # ties
    x[1, 0, 0, 0, 0], x[1, 0, 0, 0, 31] = 0, 15
    x = x.to(dtype).transpose(2, 3)
    cache = Int4KVCache(pages, H, D, page_size=P, dtype=dtype, device=device)
    start_codes = torch.randint(0, 256, cache.codes.shape, generator=g).to(torch.uint8)
    start_params = torch.randn(cache.params.shape, generator=g).to(dtype)
    cache.codes.copy_(start_codes), cache.params.copy_(start_params)
    at = (table.to(device), _int(starts, device), _int(counts, device))
    cache.append(x[0].to(device), x[1].to(device), *at)
    k, v = cache.read(*at, T)
    torch.cuda.synchronize()
    codes, params = start_codes, start_params
    for side, got in ((0, k), (1, v)):
        c, s, m = ref.quantise(x[side])
        numbers = ref.values(c, s, m).to(dtype)
        for b in range(B):
            for t in range(min(counts[b], T)):
                p, slot = table[b, (starts[b] + t) // P], (starts[b] + t) % P
                codes[side, p, :, slot] = ref.pack(c[b, :, t])
                params[side, p, :, 0, :, slot], params[side, p, :, 1, :, slot] = s[b, :, t], m[b, :, t]
            numbers[b, :, min(counts[b], T) :] = 0
        assert torch.equal(got.cpu(), numbers)
    assert torch.equal(cache.codes.cpu(), codes)
    assert torch.equal(cache.params.cpu().view(torch.int16), params.view(torch.int16))


def test_append_leaves_out_what_has_no_page(device):
    """Negative starts, positions past the table, entries that are no page, counts outside the tokens."""
    g = gen(2)
    P, H, D, T = 16, 2, 64, 40
    cache = Int4KVCache(4, H, D, page_size=P, device=device)
    cache.codes.fill_(0x5A)
    table = _int([[0, -1], [4, 1], [1 << 30, 2], [3, -(1 << 31)]], device)
    starts, counts = _int([-8, 0, 16, 30], device), _int([100, 40, 40, -7], device)
    x = torch.randn((4, H, T, D), generator=g).to(torch.bfloat16).to(device)
    cache.append(x, x, table, starts, counts)
    k, v = cache.read(table, starts, counts, T)
    torch.cuda.synchronize()
    want = torch.zeros((4, H, T, D), dtype=torch.bfloat16)
    back = ref.values(*ref.quantise(x.cpu())).to(torch.bfloat16)
    want[0, :, 8:24] = back[0, :, 8:24]  # position -8 + 8 on, page 0
    want[1, :, 16:32] = back[1, :, 16:32]  # page 1
    want[2, :, 0:16] = back[2, :, 0:16]  # page 2
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
    assert (cache.codes[:, 3] == 0x5A).all()


def _filled(device, dtype, D, H, P, lengths, seed, spare=3, spread=1.0):
    """A cache with random pasts; its pages' unused slots hold NaN parameters."""
    g = gen(seed)
    B, width = len(lengths), max(1, -(-max(lengths) // P))
    pages = B * width + spare
    table = _table(B, width, pages, g)
    cache = Int4KVCache(pages, H, D, page_size=P, dtype=dtype, device=device)
    cache.params.fill_(float("nan"))
    T = max(lengths)
    x = torch.randn((2, B, T, H, D), generator=g) * spread
    x[0] += torch.randn((1, 1, H, D), generator=g) / 2
    x = x.to(dtype).to(device).transpose(2, 3)
    cache.append(x[0], x[1], table.to(device), torch.zeros(B, dtype=torch.int32, device=device), _int(lengths, device))
    torch.cuda.synchronize()
    return cache, table, g


def _attend_check(device, cache, table, q, lengths, window=None, sinks=0, scale=None, there=None):
    got = cache.attend(q.to(device), table.to(device), _int(lengths, device), window=window, sinks=sinks, scale=scale)
    torch.cuda.synchronize()
    codes, params = cache.codes.cpu(), cache.params.cpu()
    B, Hq, Q, D = q.shape
    u = torch.finfo(q.dtype).eps / 2
    uw = 2.0**-8 if q.dtype == torch.bfloat16 else 2.0**-16 + 2.0**-24
    for b in range(B):
        n = min(max(lengths[b], 0), table.shape[1] * cache.page_size)
        k, v = (ref.sequence(codes, params, table[b].tolist(), n, side) for side in range(2))
        m = ref.sequence(torch.zeros_like(codes), params, table[b].tolist(), n, 1).abs()
        p, j = n - Q + torch.arange(Q)[:, None], torch.arange(n)[None]
        mask = (j <= p) & ((p - j < (window or n + 1)) | (j < sinks))
        if there is not None:
            mask = mask & there[b][None, :n]
        if n == 0:
            assert (got[b] == 0).all()
            continue
        G = Hq // cache.kv_heads
        kk, vv, mm = (x.repeat_interleave(G, 0) for x in (k, v, m))
        sc = D**-0.5 if scale is None else scale
        s = q[b].double() @ kk.transpose(1, 2) * sc
        # 32-bit sums: D products of numbers up to 16 + 15 steps, group by group
        es = 2.0**-24 * (D + 40) * 3 * sc * (q[b].double().abs() @ (kk.abs() + 3 * (kk - mm).abs()).transpose(1, 2)) + 2.0**-20
        s = torch.where(mask, s, -torch.inf)
        e = torch.where(mask, torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300)), 0.0)
        w = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
        ew = w * (2 * torch.where(mask, es, 0.0).amax(-1, keepdim=True) + 2.0**-18)
        out = w @ vv
        steps = (vv.abs() + mm)  # at least s c
        # f16 weights of the minima: half a step of its subnormal numbers
        low = 2.0**-25 if q.dtype == torch.float16 else 0.0
        # 16 + c and -16 cancel in 32 bits: 2^-24 of 16 steps, twice (the result can be far smaller)
        group = torch.stack([x.amax(-1) for x in (vv - mm).abs().split(32, -1)], -1).repeat_interleave(32, -1) + mm
        bound = (uw * w) @ steps + (u * w + torch.where(mask, low, 0.0)) @ mm + ew @ (vv.abs() + 4 * group)
        bound = bound + 2.0**-22 * 16 * (w @ group) + u * out.abs() + 2.0**-24 * u + 1e-30
        attn.assert_within(got[b], out, bound, f"sequence {b}")
    return got


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("Hq,H,Q,P,lengths,window,sinks", [
    (2, 1, 1, 16, [1, 2, 15, 16, 17, 31, 32, 33], None, 0), (4, 4, 1, 32, [64, 65, 100, 0], None, 0),
    (8, 2, 1, 64, [700, 513, 1], None, 0), (14, 2, 5, 16, [300, 5, 4, 3], 100, 3), (3, 1, 2, 48, [97, 200], 1, 0),
    (16, 1, 8, 128, [400, 131], 33, 2), (6, 2, 3, 256, [600, 40], 64, 70), (4, 2, 1, 64, [1500, 900], 128, 4),
    (2, 2, 1, 64, [3000], 40, 0), (2, 1, 17, 16, [130, 16], None, 0),
])
def test_attend(device, dtype, D, Hq, H, Q, P, lengths, window, sinks):
    cache, table, g = _filled(device, dtype, D, H, P, lengths, seed=sum(lengths))
    q = torch.randn((len(lengths), Q, Hq, D), generator=g).to(dtype).transpose(1, 2)
    _attend_check(device, cache, table, q, lengths, window, sinks)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("spread,size", [(1e-3, 1.0), (100.0, 0.05), (1.0, 8.0)])
def test_attend_small_large_and_sharp(device, dtype, D, spread, size):
    cache, table, g = _filled(device, dtype, D, 2, 32, [500, 77], seed=5, spread=spread)
    q = (torch.randn((2, 4, 1, D), generator=g) * size).to(dtype)
    _attend_check(device, cache, table, q, [500, 77], scale=0.1)


def test_attend_leaves_out_what_has_no_page(device):
    """Entries that are no page, lengths past the table and below zero."""
    P, D = 32, 128
    cache, table, g = _filled(device, torch.bfloat16, D, 2, P, [200, 200, 200, 200], seed=7)
    there = torch.ones((4, 7 * P), dtype=torch.bool)
    for b, i, bad in ((0, 1, -1), (1, 0, cache.pages), (1, 6, 1 << 30), (2, 3, -(1 << 31))):
        table[b, i] = bad
        there[b, i * P : (i + 1) * P] = False
    for i in range(7):
        table[3, i] = -5
    there[3] = False
    q = torch.randn((4, 4, 2, D), generator=g).to(torch.bfloat16)
    got = _attend_check(device, cache, table, q, [200, 200, 200, 200], there=there)
    assert (got[3] == 0).all()
    got = cache.attend(q.to(device), table.to(device), _int([-3, 0, 2**31 - 1, 9], device))
    torch.cuda.synchronize()
    assert (got[:2] == 0).all()


def test_attend_long_is_split_and_joined(device):
    """A long past of one sequence, in workgroups of their own, the same on every call and on another stream."""
    n, P, D = 20000, 64, 64
    cache, table, g = _filled(device, torch.bfloat16, D, 1, P, [n], seed=8)
    q = torch.randn((1, 2, 1, D), generator=g).to(torch.bfloat16)
    got = _attend_check(device, cache, table, q, [n])
    args = (q.to(device), table.to(device), _int([n], device))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = cache.attend(*args)
    torch.cuda.synchronize()
    assert torch.equal(got, again)


def test_decode_steps_in_a_graph(device):
    """Append, read and attend of one step captured; tables, lengths and inputs change between replays."""
    P, H, D, B = 16, 2, 128, 3
    cache, table, g = _filled(device, torch.bfloat16, D, H, P, [50, 20, 90], seed=9)
    twin = Int4KVCache(cache.pages, H, D, page_size=P, device=device)
    twin.codes.copy_(cache.codes), twin.params.copy_(cache.params)
    table = table.to(device)
    lengths = _int([51, 21, 91], device)
    one = torch.ones(B, dtype=torch.int32, device=device)
    x = torch.randn((3, B, 4, 1, D), generator=g).to(torch.bfloat16).to(device)

    def step(c):
        c.append(x[0][:, :H], x[1][:, :H], table, lengths - 1, one)
        return (*c.read(table, lengths - 1, one, 1), c.attend(x[2], table, lengths, window=60, sinks=2))

    step(twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=g))
        want = step(twin)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        lengths.add_(1)


def test_offsets_past_32_bits(device):
    """The far pages of a cache whose sides are more than 2 GiB each, as a small cache's."""
    P, H, D, far = 4096, 2, 64, 9000
    big = Int4KVCache(far, H, D, page_size=P, device=device)
    small = Int4KVCache(3, H, D, page_size=P, device=device)
    assert big.codes[0].numel() > 1 << 31
    g = gen(12)
    x = torch.randn((2, 1, H, 5000, D), generator=g).to(torch.bfloat16).to(device)
    q = torch.randn((1, 4, 2, D), generator=g).to(torch.bfloat16).to(device)
    starts, counts, lengths = _int([100], device), _int([5000], device), _int([5100], device)
    results = []
    for cache, pages in ((big, [far - 1, 4321]), (small, [0, 2])):
        table = _int([pages], device)
        cache.append(x[0], x[1], table, starts, counts)
        results.append((*cache.read(table, starts, counts, 5000), cache.attend(q, table, lengths, window=4500)))
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][0].abs().amax(-1).min() > 0


def test_strides_of_inputs(device):
    """Slices of a fused projection, unaligned and transposed inputs: as their copies."""
    P, H, D = 16, 2, 64
    cache, table, g = _filled(device, torch.float16, D, H, P, [60, 60], seed=10)
    fused = torch.randn((2, 3, 4 + 2 * H, D), generator=g).half().to(device)
    q, k, v = (fused[:, :, i:j].transpose(1, 2) for i, j in ((0, 4), (4, 4 + H), (4 + H, 4 + 2 * H)))
    at = (table.to(device), _int([50, 45], device), _int([3, 2], device))
    lengths = _int([53, 47], device)
    results = []
    odd = lambda t: torch.empty(t.numel() + 3, dtype=t.dtype, device=device)[3:].view(t.shape).copy_(t)
    for form in (lambda t: t, torch.Tensor.contiguous, odd, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        cache.append(form(k), form(v), *at)
        results.append((cache.codes.clone(), cache.attend(form(q), at[0], lengths)))
    for r in results[1:]:
        assert torch.equal(r[0], results[0][0]) and torch.equal(r[1], results[0][1])


def test_nothing_to_do(device):
    cache = Int4KVCache(2, 1, 64, page_size=16, device=device)
    none = torch.zeros((0, 1), dtype=torch.int32, device=device)
    empty = torch.zeros(0, dtype=torch.int32, device=device)
    x = torch.zeros((0, 1, 3, 64), dtype=torch.bfloat16, device=device)
    cache.append(x, x, none, empty, empty)
    assert cache.read(none, empty, empty, 3)[0].shape == x.shape
    assert cache.attend(x, none, empty).shape == x.shape
    table, n = torch.zeros((1, 0), dtype=torch.int32, device=device), _int([5], device)
    one = torch.ones((1, 1, 2, 64), dtype=torch.bfloat16, device=device)
    assert (cache.attend(one, table, n) == 0).all()
    cache.append(one, one, table, n, n)
    assert (cache.read(table, n, n, 2)[0] == 0).all()
    assert cache.attend(one[:, :, :0], table, n).shape == (1, 1, 0, 64)
