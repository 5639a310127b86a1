"""Timed cases of the attention beside the memories: window attention, the 4-bit key / value cache, attention over it.

listed() names the cases, draw() gives more of the same ranges, prepare() makes
a case's inputs on the GPU from a seed, run() takes one pass: where `own` is
true through the framework's entry points, else through plain torch operations
in 32 bits. exact() computes the same outputs from the definitions in 64 bits
and work() says what a pass cannot do without.

Key j is visible to the query at position p of a sequence of tokens
[start, end) if start <= j <= p < end and (p - j < window or j - start < sinks);
window 0 stands for no window.

The 4-bit cache holds each key / value head vector in groups of 32 numbers:
minimum m and step s = (max - min) / 15 in the cache's type, codes
c = round((x - m) / s), the number read back is m + s c. Of the codes of one
vector, number d = lane + 16 i (lane < 16) lies at: head 64, 16-bit word
`lane`, bits 4 i; head 128, 32-bit word `lane`, bits 4 (i / 2 + 4 (i % 2)).
codes: [2 (K, V), pages, heads, page, head / 2] bytes;
params: [2 (K, V), pages, heads, 2 (s, m), head / 32, page] of the cache's type.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 32


def listed():
    return [
        # The smallest training call: one short sequence of the decoder benchmark's heads, forward and backward.
        {"name": "train_short", "op": "train", "batch": 1, "seq": 192, "q_heads": 16, "kv_heads": 8, "dim": 128,
         "window": 128, "sinks": 4, "pad": "none", "dtype": "bf16"},
        # A training step's attention at the decoder benchmark's heads and its longest sequence.
        {"name": "train_window", "op": "train", "batch": 4, "seq": 4096, "q_heads": 16, "kv_heads": 8, "dim": 128,
         "window": 1024, "sinks": 4, "pad": "none", "dtype": "bf16"},
        # A padded batch of odd length and small heads, no sharing of key heads, no window, 16-bit floats.
        {"name": "train_ragged_f16", "op": "train", "batch": 3, "seq": 1777, "q_heads": 12, "kv_heads": 12, "dim": 64,
         "window": 0, "sinks": 0, "pad": "right", "dtype": "f16"},
        # A long prompt, forward alone.
        {"name": "prompt_long", "op": "prompt", "batch": 1, "seq": 32768, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "window": 4096, "sinks": 8, "pad": "none", "dtype": "bf16"},
        # Prompts of several lengths as generation pads them, on the left.
        {"name": "prompt_left", "op": "prompt", "batch": 8, "seq": 777, "q_heads": 16, "kv_heads": 8, "dim": 128,
         "window": 256, "sinks": 4, "pad": "left", "dtype": "bf16"},
        # One new token of each of 64 sequences is quantised into its page and read back.
        {"name": "store_tokens", "op": "store", "batch": 64, "tokens": 1, "at": 4000, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
        # Prompts of several lengths are written into the cache and read back.
        {"name": "store_prompts", "op": "store", "batch": 8, "tokens": 5000, "at": 0, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
        # A single sequence answers, a token at a time, from a short cache.
        {"name": "decode_one", "op": "decode", "batch": 1, "queries": 1, "length": 1000, "q_heads": 16, "kv_heads": 8,
         "dim": 128, "window": 0, "sinks": 0, "page": 64, "dtype": "bf16"},
        # A single sequence with a long past, all of it visible.
        {"name": "decode_long", "op": "decode", "batch": 1, "queries": 1, "length": 131072, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "page": 64, "dtype": "bf16"},
        # A serving batch of ragged lengths.
        {"name": "decode_batch", "op": "decode", "batch": 64, "queries": 1, "length": 16000, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "page": 64, "dtype": "bf16"},
        # The same through a window with sinks.
        {"name": "decode_window", "op": "decode", "batch": 64, "queries": 1, "length": 16000, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4, "page": 64, "dtype": "bf16"},
        # A few drafted tokens at once, small pages and heads, 16-bit floats.
        {"name": "decode_draft_f16", "op": "decode", "batch": 16, "queries": 5, "length": 3001, "q_heads": 14,
         "kv_heads": 2, "dim": 64, "window": 2000, "sinks": 3, "page": 16, "dtype": "f16"},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


HEADS = [(16, 8), (16, 8), (32, 8), (8, 8), (12, 12), (14, 2), (6, 2), (16, 1), (24, 8)]


def draw(rng):
    top = [work(case) for case in listed()]
    while True:
        case = _drawn(rng)
        cost = work(case)
        if all(cost[n] <= max(w[n] for w in top) for n in cost):
            return case


def _drawn(rng):
    op = rng.choice(["train", "train", "prompt", "prompt", "store", "decode", "decode", "decode"])
    q_heads, kv_heads = rng.choice(HEADS)
    case = {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]),
            "dtype": rng.choice(["bf16", "bf16", "f16"])}
    window = rng.choice([0, _between(rng, 16, 4096), _between(rng, 16, 4096)])
    sinks = 0 if window == 0 else rng.choice([0, 1, 4, rng.randint(2, 64)])
    if op in ("train", "prompt"):
        seq = _between(rng, 1, 8192 if op == "train" else 32768)
        if seq > 8192 and window == 0:
            window = 4096
        case.update(batch=rng.randint(1, max(1, min(8, 16384 // seq))), seq=seq, window=window, sinks=sinks,
                    pad=rng.choice(["none", "left", "right"]))
        return case
    if op == "store":
        del case["q_heads"]
        tokens = rng.choice([1, _between(rng, 1, 8192)])
        case.update(batch=_between(rng, 1, 64 if tokens == 1 else max(1, min(64, 40000 // tokens))), tokens=tokens,
                    at=_between(rng, 1, 8192), page=rng.choice([16, 32, 64, 128]))
        return case
    length = _between(rng, 1, 131072)
    case.update(batch=_between(rng, 1, max(1, min(128, 1000000 // length))), queries=rng.choice([1, 1, 1, rng.randint(2, 8)]),
                length=length, window=window, sinks=sinks, page=rng.choice([16, 32, 64, 128, 256]))
    return case


def _spread(case, n):
    """The sequences' lengths: the first is whole, the others fall evenly towards a quarter of it."""
    B = case["batch"]
    return [max(1, n - (b * n * 3) // (4 * B)) for b in range(B)]


def _bounds(case):
    """(start, end) of each sequence of a padded batch."""
    T, pad = case["seq"], case["pad"]
    if pad == "none":
        return [(0, T)] * case["batch"]
    return [(T - n, T) if pad == "left" else (0, n) for n in _spread(case, T)]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _heads(gen, B, T, H, D, dtype, offset=0.0):
    """[B, H, T, D] as a projection leaves it: a view of [B, T, H, D]. Keys have channels of their own mean."""
    x = torch.randn((B, T, H, D), generator=gen, device="cuda")
    if offset:
        x += offset * torch.randn((1, 1, H, D), generator=gen, device="cuda")
    return x.to(dtype).transpose(1, 2)


def _pages(gen, B, width, page_count):
    """A page table [B, width] of distinct pages in no order."""
    return torch.randperm(page_count, generator=gen, device="cuda")[: B * width].view(B, width).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, Hk, D = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["op"] in ("train", "prompt"):
        B, T, Hq = case["batch"], case["seq"], case["q_heads"]
        state["q"] = _heads(gen, B, T, Hq, D, dtype)
        state["k"] = _heads(gen, B, T, Hk, D, dtype, 0.5)
        state["v"] = _heads(gen, B, T, Hk, D, dtype)
        if case["op"] == "train":
            state["do"] = _heads(gen, B, T, Hq, D, dtype)
        if case["pad"] != "none":
            bounds = torch.tensor(_bounds(case), dtype=torch.int32, device="cuda")
            state["starts"], state["ends"] = bounds[:, 0].contiguous(), bounds[:, 1].contiguous()
        if own:
            for name in ("q", "k", "v"):
                state[name].requires_grad_(case["op"] == "train")
        return state
    B, P = case["batch"], case["page"]
    if case["op"] == "store":
        T, at = case["tokens"], case["at"]
        width = -(-(at + T) // P)
        state["k"] = _heads(gen, B, T, Hk, D, dtype, 0.5)
        state["v"] = _heads(gen, B, T, Hk, D, dtype)
        state["starts"] = torch.full((B,), at, dtype=torch.int32, device="cuda")
        state["counts"] = torch.tensor(_spread(case, T), dtype=torch.int32, device="cuda")
    else:
        lengths = _spread(case, case["length"])
        width = -(-case["length"] // P)
        state["q"] = _heads(gen, B, case["queries"], case["q_heads"], D, dtype)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    pages = B * width + 3
    state["table"] = _pages(gen, B, width, pages)
    codes = torch.zeros((2, pages, Hk, P, D // 2), dtype=torch.uint8, device="cuda")
    params = torch.zeros((2, pages, Hk, 2, D // GROUP, P), dtype=dtype, device="cuda")
    if case["op"] == "decode":  # the past, quantised page by page
        mean = 0.5 * torch.randn((1, Hk, 1, D), generator=gen, device="cuda")
        step = max(1, (1 << 26) // (Hk * P * D))
        for side in range(2):
            for p0 in range(0, pages, step):
                n = min(step, pages - p0)
                x = torch.randn((n, Hk, P, D), generator=gen, device="cuda")
                c, s, m = _quantise((x + mean if side == 0 else x).to(dtype))
                codes[side, p0 : p0 + n] = _pack(c)
                params[side, p0 : p0 + n, :, 0] = s.transpose(-1, -2)
                params[side, p0 : p0 + n, :, 1] = m.transpose(-1, -2)
    if own:
        from modelos_amd.kv_cache import Int4KVCache

        state["cache"] = Int4KVCache(pages, Hk, D, page_size=P, dtype=dtype, device="cuda")
        state["cache"].codes.copy_(codes)
        state["cache"].params.copy_(params)
    else:
        state["codes"], state["params"] = codes, params
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return {"train": _plain_window, "prompt": _plain_window, "store": _plain_store,
                "decode": _plain_decode}[case["op"]](state)
    window = case.get("window") or None
    if case["op"] in ("train", "prompt"):
        from modelos_amd.window_attention import window_attention

        q, k, v = state["q"], state["k"], state["v"]
        out = window_attention(q, k, v, window=window, sinks=case["sinks"], starts=state.get("starts"),
                               ends=state.get("ends"))
        if case["op"] == "prompt":
            return out
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), state["do"])]
    cache, table = state["cache"], state["table"]
    if case["op"] == "store":
        cache.append(state["k"], state["v"], table, state["starts"], state["counts"])
        return list(cache.read(table, state["starts"], state["counts"], case["tokens"]))
    return cache.attend(state["q"], table, state["lengths"], window=window, sinks=case["sinks"])


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_sequence(q, k, v, W, S, do):
    """One sequence, all of it tokens: q, do [Hq, n, D], k, v [Hk, n, D], 32 bits. Blocks of queries against the keys
    that the block can see. Returns o, or o and the three gradients."""
    Hq, n, D = q.shape
    Hk = k.shape[0]
    G, scale = Hq // Hk, D**-0.5
    W = W or n
    q = q.view(Hk, G, n, D)
    o = torch.empty_like(q)
    if do is not None:
        do = do.view(Hk, G, n, D)
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    block = 1024
    for i0 in range(0, n, block):
        i1 = min(n, i0 + block)
        lo = max(0, i0 - W + 1)
        first = min(S, lo)
        cols = torch.cat([torch.arange(first, device=q.device), torch.arange(lo, i1, device=q.device)])
        rows = torch.arange(i0, i1, device=q.device)[:, None]
        hidden = (cols > rows) | ((rows - cols >= W) & (cols >= S))
        kk, vv = torch.cat([k[:, :first], k[:, lo:i1]], 1), torch.cat([v[:, :first], v[:, lo:i1]], 1)
        qq = q[:, :, i0:i1].reshape(Hk, -1, D)
        s = torch.matmul(qq, kk.transpose(1, 2)).mul_(scale).view(Hk, G, i1 - i0, -1)
        s.masked_fill_(hidden, -math.inf)
        p = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
        p = (p / p.sum(-1, keepdim=True)).view(Hk, G * (i1 - i0), -1)
        oo = torch.matmul(p, vv)
        o[:, :, i0:i1] = oo.view(Hk, G, i1 - i0, D)
        if do is None:
            continue
        dd = do[:, :, i0:i1].reshape(Hk, -1, D)
        ds = torch.matmul(dd, vv.transpose(1, 2)).sub_((dd * oo).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dq[:, :, i0:i1] = torch.matmul(ds, kk).view(Hk, G, i1 - i0, D)
        dkk, dvv = torch.matmul(ds.transpose(1, 2), qq), torch.matmul(p.transpose(1, 2), dd)
        dk[:, :first] += dkk[:, :first]
        dk[:, lo:i1] += dkk[:, first:]
        dv[:, :first] += dvv[:, :first]
        dv[:, lo:i1] += dvv[:, first:]
    if do is None:
        return (o.view(Hq, n, D),)
    return o.view(Hq, n, D), dq.view(Hq, n, D), dk, dv


def _plain_window(state):
    case = state["case"]
    names = ("q", "k", "v") + (("do",) if case["op"] == "train" else ())
    x = [state[name] for name in names]
    train = case["op"] == "train"
    outs = [torch.zeros_like(t) for t in ([x[0], x[0], x[1], x[2]] if train else [x[0]])]
    for b, (i, j) in enumerate(_bounds(case)):
        part = [t[b, :, i:j].float().contiguous() for t in x]
        got = _plain_sequence(*part[:3], case["window"], case["sinks"], part[3] if train else None)
        for out, g in zip(outs, got):
            out[b, :, i:j] = g.to(out.dtype)
    return outs if train else outs[0]


def _quantise(x):
    """Codes [..., D], steps and minima [..., D / 32] of x [..., D]."""
    g = x.unflatten(-1, (-1, GROUP)).float()
    m, top = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((top - m) / 15).to(x.dtype).float()
    c = torch.where(s > 0, torch.round((g - m) / torch.where(s > 0, s, 1)), 0).clamp(0, 15)
    return c.flatten(-2).to(torch.uint8), s.squeeze(-1).to(x.dtype), m.squeeze(-1).to(x.dtype)


def _pack(c):
    """Bytes [..., D / 2] of codes [..., D]."""
    if c.shape[-1] == 64:  # (byte, nibble, lane) of number lane + 16 (2 byte + nibble)
        c = c.unflatten(-1, (2, 2, 16)).movedim(-1, -3)
    else:  # (byte % 2, nibble, byte / 2, lane)
        c = c.unflatten(-1, (2, 2, 2, 16)).movedim((-1, -2, -4, -3), (-4, -3, -2, -1)).flatten(-3, -2)
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-2)


def _unpack(b, D):
    """Codes [..., D] of bytes [..., D / 2]."""
    if D == 64:
        b = b.unflatten(-1, (16, 2))
        return torch.stack([b & 15, b >> 4], -1).movedim(-3, -1).flatten(-3)
    b = b.unflatten(-1, (16, 2, 2))
    return torch.stack([b & 15, b >> 4], -1).movedim((-4, -3, -2, -1), (-1, -2, -4, -3)).flatten(-4)


def _numbers(codes, params, page, slot, D):
    """The numbers of tokens (page, slot) [N] in 32 bits: [N, heads, D]."""
    c = _unpack(codes[page, :, slot], D).float().unflatten(-1, (-1, GROUP))
    p = params[page, :, :, :, slot].float()
    return (c * p[:, :, 0, :, None] + p[:, :, 1, :, None]).flatten(-2)


def _plain_store(state):
    case, codes, params = state["case"], state["codes"], state["params"]
    T, D, P, B = case["tokens"], case["dim"], case["page"], case["batch"]
    at = torch.arange(T, device="cuda")
    live = (at < state["counts"][:, None]).flatten()
    place = state["starts"][:, None] + at
    page = torch.gather(state["table"].long(), 1, (place // P).long()).flatten()[live]
    slot = (place % P).long().flatten()[live]
    outs = []
    for side, name in enumerate(("k", "v")):
        x = state[name].transpose(1, 2).flatten(0, 1)[live]
        c, s, m = _quantise(x)
        codes[side][page, :, slot] = _pack(c)
        params[side][page, :, 0, :, slot] = s
        params[side][page, :, 1, :, slot] = m
        back = torch.zeros((B * T, x.shape[1], D), dtype=x.dtype, device="cuda")
        back[live] = _numbers(codes[side], params[side], page, slot, D).to(x.dtype)
        outs.append(back.view(B, T, -1, D).transpose(1, 2))
    return outs


def _plain_decode(state):
    case, codes, params, table = state["case"], state["codes"], state["params"], state["table"]
    B, Q, Hq, Hk, D, P = (case[n] for n in ("batch", "queries", "q_heads", "kv_heads", "dim", "page"))
    W, S, top = case["window"] or (1 << 30), case["sinks"], case["length"]
    out = torch.empty((B, Hq, Q, D), dtype=state["q"].dtype, device="cuda")
    span = min(top, W + Q - 1)
    first = min(S, top)
    step = max(1, (1 << 29) // ((first + span) * Hk * D))
    for b in range(0, B, step):
        n = state["lengths"][b : b + step].long()[:, None]
        near = torch.arange(-span, 0, device="cuda") + n
        j = torch.cat([torch.arange(first, device="cuda").expand(n.shape[0], -1), near], 1)
        there = (j >= 0) & (j < n)
        there[:, first:] &= near >= first
        at = j.clamp(0, top - 1)
        page, slot = torch.gather(table[b : b + step].long(), 1, at // P).flatten(), (at % P).flatten()
        k, v = (_numbers(codes[i], params[i], page, slot, D).view(*j.shape, Hk, D).transpose(1, 2).contiguous()
                for i in range(2))
        q = state["q"][b : b + step].float().reshape(-1, Hk, Hq // Hk * Q, D)
        s = torch.matmul(q, k.transpose(2, 3)).mul_(D**-0.5).unflatten(2, (-1, Q))
        p = (n - Q + torch.arange(Q, device="cuda"))[:, :, None]  # [b, Q, 1]
        seen = there[:, None] & (p >= 0) & (j[:, None] <= p) & ((p - j[:, None] < W) | (j[:, None] < S))
        s.masked_fill_(~seen[:, None, None], -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
        e = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
        out[b : b + step] = torch.matmul(e.flatten(2, 3), v).view(-1, Hq, Q, D).to(out.dtype)
    return out


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _attention64(q, k, v, position, key_position, W, S, do=None):
    """One head: softmax over the keys each query sees, [nq, D], [nk, D]; with do the three gradients too."""
    q, k, v = q.double(), k.double(), v.double()
    scale = 1 / math.sqrt(q.shape[1])
    gap = position[:, None] - key_position[None, :]
    seen = (gap >= 0) & (position[:, None] >= 0)
    if W:
        seen &= (gap < W) | (key_position[None, :] < S)
    logits = torch.where(seen, q @ k.T * scale, -math.inf)
    weights = torch.where(seen.any(1, keepdim=True), torch.softmax(logits, 1), 0.0)
    o = weights @ v
    if do is None:
        return (o,)
    do = do.double()
    d_weights = do @ v.T
    d_logits = weights * (d_weights - (d_weights * weights).sum(1, keepdim=True))
    return o, d_logits @ k * scale, d_logits.T @ q * scale, weights.T @ do


def _value64(case, codes, params, table, b, head, side, n):
    """Numbers [n, D] of a sequence's first n tokens of one head, code by code."""
    D, P = case["dim"], case["page"]
    t = torch.arange(n, device="cuda")
    page = table[b].long()[t // P]
    words = codes[side][page, head, t % P].long()
    d = torch.arange(D, device="cuda")
    lane, i = d % 16, d // 16
    bit = 16 * lane + 4 * i if D == 64 else 32 * lane + 4 * (i // 2 + 4 * (i % 2))
    c = (words[:, bit // 8] >> (bit % 8)) & 15
    par = params[side][page, head, :, :, t % P].double()
    return c.double() * par[:, 0][:, d // GROUP] + par[:, 1][:, d // GROUP]


def exact(case, seed):
    state = prepare(case, seed)
    W, S = case.get("window"), case.get("sinks")
    if case["op"] in ("train", "prompt"):
        x = [state[n].detach() for n in ("q", "k", "v")]
        do = state.get("do")
        shapes = [x[0], x[0], x[1], x[2]] if do is not None else [x[0]]
        outs = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in shapes]
        share = case["q_heads"] // case["kv_heads"]
        for b, (i, j) in enumerate(_bounds(case)):
            key_at = torch.arange(j - i, device="cuda")
            for h in range(case["q_heads"]):
                for r in range(0, j - i, 2048):  # rows of queries, against every key up to the last one's
                    e = min(r + 2048, j - i)
                    rows = slice(i + r, i + e)
                    got = _attention64(x[0][b, h, rows], x[1][b, h // share, i : i + e], x[2][b, h // share, i : i + e],
                                       key_at[r:e], key_at[:e], W, S, None if do is None else do[b, h, rows])
                    outs[0][b, h, rows] = got[0]
                    if do is not None:
                        outs[1][b, h, rows] = got[1]
                        outs[2][b, h // share, i : i + e] += got[2]
                        outs[3][b, h // share, i : i + e] += got[3]
        return outs if do is not None else outs[0]
    if case["op"] == "store":
        outs = []
        for name in ("k", "v"):
            x = state[name].double().unflatten(-1, (-1, GROUP))
            low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
            s = ((high - low) / 15).to(state[name].dtype).double()
            c = torch.round((x - low) / s.clamp_min(1e-300)).clamp(0, 15)
            x = torch.where(s > 0, low + c * s, low).flatten(-2)
            keep = torch.arange(x.shape[2], device="cuda")[None] < state["counts"][:, None]
            outs.append(x * keep[:, None, :, None])
        return outs
    codes, params, table = (state["cache"].codes, state["cache"].params, state["table"]) if own else (
        state["codes"], state["params"], state["table"])
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    share = case["q_heads"] // case["kv_heads"]
    for b, n in enumerate(state["lengths"].tolist()):
        position = n - case["queries"] + torch.arange(case["queries"], device="cuda")
        for g in range(case["kv_heads"]):
            k, v = (_value64(case, codes, params, table, b, g, side, n) for side in range(2))
            for h in range(g * share, (g + 1) * share):
                out[b, h] = _attention64(state["q"][b, h], k, v, position, torch.arange(n, device="cuda"), W, S)[0]
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _seen(n, first, W, S):
    """Visible pairs of the queries at positions [first, n) of a sequence of n tokens."""
    total = 0
    W = W or n
    for p in range(max(0, first), n):
        total += min(p + 1, W) + min(S, max(0, p + 1 - W))
    return total


def work(case):
    D, Hk = case["dim"], case["kv_heads"]
    if case["op"] in ("train", "prompt"):
        Hq, train = case["q_heads"], case["op"] == "train"
        pairs = sum(_seen(j - i, 0, case["window"], case["sinks"]) for i, j in _bounds(case))
        numbers = case["batch"] * case["seq"] * D * ((4 * Hq + 4 * Hk) if train else (2 * Hq + 2 * Hk))
        return {"bytes": 2 * numbers, "flops": (14 if train else 4) * D * Hq * pairs}
    token = 2 * Hk * (D // 2 + 4 * (D // GROUP))  # both sides of one token in the cache
    if case["op"] == "store":
        written = sum(_spread(case, case["tokens"]))
        return {"bytes": written * (4 * Hk * D + token) + case["batch"] * case["tokens"] * 4 * Hk * D,
                "flops": 12 * Hk * D * written}
    Q, Hq, W, S = case["queries"], case["q_heads"], case["window"], case["sinks"]
    tokens = pairs = 0
    for n in _spread(case, case["length"]):
        near = min(n, (W or n) + Q - 1)
        tokens += near + min(S, n - near)
        pairs += _seen(n, n - Q, W, S)
    return {"bytes": tokens * token + 4 * case["batch"] * Q * Hq * D, "flops": 4 * D * Hq * pairs}
