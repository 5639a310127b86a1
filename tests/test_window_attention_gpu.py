"""Window attention with sinks (modelos_amd.window_attention) against the formulas in 64 bits, forward and backward.

Bounds (oracle.attention): a rounding to 16 bits is off by at most u = eps / 2 of its value; weights, their gradients
and results are each rounded once, everything else is summed in 32 bits."""
from __future__ import annotations

import pytest
import torch

from modelos_amd.window_attention import window_attention
from oracle import attention as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _inputs(B, T, H, Hk, D, dtype, seed=0, grad_scale=1.0):
    g = gen(seed)
    make = lambda h: torch.randn((B, T, h, D), generator=g).to(dtype).transpose(1, 2)
    q, k, v, do = make(H), make(Hk), make(Hk), make(H)
    return q, k + torch.randn((1, Hk, 1, D), generator=g).to(dtype) / 2, v, (do.float() * grad_scale).to(dtype)


def _run(device, q, k, v, do, **kw):
    x = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    for name in ("starts", "ends"):
        if kw.get(name) is not None:
            kw[name] = torch.tensor(kw[name], dtype=torch.int32, device=device)
    out = window_attention(*x, **kw)
    grads = torch.autograd.grad(out, x, do.to(device))
    torch.cuda.synchronize()
    return [out.detach(), *grads]


def _check(device, q, k, v, do, window=None, sinks=0, starts=None, ends=None, scale=None):
    got = _run(device, q, k, v, do, window=window, sinks=sinks, starts=starts, ends=ends, scale=scale)
    mask = ref.masks(q.shape[0], q.shape[2], window, sinks, starts, ends)
    values, bounds = ref.attention(q, k, v, mask, scale, do)
    for name, g, e, b, like in zip(("out", "dq", "dk", "dv"), got, values, bounds, (q, q, k, v)):
        assert g.dtype == like.dtype
        ref.assert_within(g, e, b, name)
    return got


TYPES = [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64)]
TYPE_IDS = ["bf16-128", "bf16-64", "f16-128", "f16-64"]


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("T,H,Hk,window,sinks", [
    (1, 2, 1, None, 0), (2, 4, 4, None, 0), (5, 4, 1, 1, 0), (63, 3, 1, None, 0), (64, 2, 2, 7, 1), (65, 4, 2, 64, 0),
    (129, 6, 3, 33, 5), (200, 8, 2, 64, 4), (257, 5, 1, 100, 70), (321, 2, 1, 20, 2), (300, 2, 1, 1000, 3),
    (190, 4, 1, 30, 190), (450, 2, 2, 16, 130), (1030, 1, 1, 129, 9),
])
def test_lengths_and_windows(device, dtype, D, T, H, Hk, window, sinks):
    _check(device, *_inputs(2 if T < 400 else 1, T, H, Hk, D, dtype, seed=T), window, sinks)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (17, 0), (40, 3)])
def test_padding_is_not_used(device, dtype, D, window, sinks):
    """Left, right and both pads, an empty sequence, bounds outside the tokens; padding holds NaN and infinities."""
    T = 150
    starts, ends = [0, 37, 0, 70, 149, -5, 90], [150, 150, 64, 133, 150, 1000, 80]
    q, k, v, do = _inputs(len(starts), T, 4, 2, D, dtype, seed=3)
    for b in range(len(starts)):
        pad = torch.ones(T, dtype=torch.bool)
        pad[max(starts[b], 0) : max(ends[b], 0)] = False
        for i, x in enumerate((q, k, v, do)):
            x[b][:, pad] = (NAN, float("inf"), NAN, -float("inf"))[i]
    got = _check(device, q, k, v, do, window, sinks, starts, ends)
    for g in got:
        assert (g[6] == 0).all() and (g[1, :, :37] == 0).all() and (g[2, :, 64:] == 0).all()


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("window,sinks", [(30, 40), (64, 3), (1, 1)])
def test_sinks_of_padded_long_sequences(device, dtype, D, window, sinks):
    """Sinks whose far queries have workgroups of their own, in sequences that start and end anywhere."""
    starts, ends = [0, 101, 0, 250, 500], [600, 600, 333, 290, 600]
    q, k, v, do = _inputs(len(starts), 600, 4, 2, D, dtype, seed=17)
    for b in range(len(starts)):
        for x in (q, k, v, do):
            x[b, :, : starts[b]] = NAN
            x[b, :, ends[b] :] = NAN
    _check(device, q, k, v, do, window, sinks, starts, ends)


@pytest.mark.parametrize("dtype,D", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (530, 2)])
def test_long_windows(device, dtype, D, window, sinks):
    """Windows that are too long for the output's rounding to be kept."""
    _check(device, *_inputs(1, 620, 2, 1, D, dtype, seed=18), window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_strides(device, dtype):
    """Heads inside a fused projection, contiguous, expanded, unaligned and sliced: the same numbers every time."""
    B, T, H, Hk, D = 2, 77, 4, 2, 64
    g = gen(5)
    fused = torch.randn((B, T, H + 2 * Hk, D), generator=g).to(dtype).to(device)
    q, k, v = (fused[:, :, i:j].transpose(1, 2) for i, j in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    do = torch.randn((B, H, T, D), generator=g).to(dtype).to(device)
    want = _run(device, q, k, v, do, window=20, sinks=2)
    mask = ref.masks(B, T, 20, 2)
    for got, e, b in zip(want, *ref.attention(q.cpu(), k.cpu(), v.cpu(), mask, None, do.cpu())):
        ref.assert_within(got, e, b)
    odd = lambda t: torch.empty(t.numel() + 3, dtype=dtype, device=device)[3:].view(t.shape).copy_(t)
    wide = lambda t: torch.empty((*t.shape[:3], 2 * D + 8), dtype=dtype, device=device)[..., :D].copy_(t)
    back = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    for form in (torch.Tensor.contiguous, odd, wide, back):
        for a, b in zip(_run(device, form(q), form(k), form(v), form(do), window=20, sinks=2), want):
            assert torch.equal(a, b)
    # one gradient for every row, one key head expanded over two
    one = do[:, :, :1].expand(B, H, T, D)
    for a, b in zip(_run(device, q, k, v, one, window=20), _run(device, q, k, v, one.contiguous(), window=20)):
        assert torch.equal(a, b)
    both = k[:, :1].expand(B, Hk, T, D)
    for a, b in zip(_run(device, q, both, v, do), _run(device, q, both.contiguous(), v, do)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", [0.01, 6.0])
def test_flat_and_sharp_logits(device, dtype, size):
    q, k, v, do = _inputs(1, 200, 2, 1, 128, dtype, seed=9)
    _check(device, (q.float() * size).to(dtype), (k.float() * size).to(dtype), v, do, 90, 4, scale=0.11)


@pytest.mark.parametrize("grad_scale", [2.0**-12, 1.0, 2.0**9])
def test_small_and_large_gradients_f16(device, grad_scale):
    """Gradients of a 16-bit float step may lie far from 1; their bounds scale with them."""
    q, k, v, do = _inputs(1, 333, 4, 2, 64, torch.float16, seed=11)
    got = _run(device, q, k, v, (do.float() * grad_scale).half(), window=200, sinks=4)
    values, bounds = ref.attention(q, k, v, ref.masks(1, 333, 200, 4), None, do)
    tiny = 2.0**-25  # a result's own subnormal rounding
    for i, name in ((1, "dq"), (2, "dk"), (3, "dv")):
        ref.assert_within(got[i], values[i] * grad_scale, bounds[i] * grad_scale + tiny, name)


def test_against_differences(device):
    """The gradients along random directions against differences of the 64-bit form."""
    q, k, v, do = _inputs(2, 90, 4, 2, 64, torch.bfloat16, seed=13)
    kw = dict(window=31, sinks=2, starts=[0, 11], ends=[90, 80])
    got = _run(device, q, k, v, do, **kw)
    mask = ref.masks(2, 90, kw["window"], kw["sinks"], kw["starts"], kw["ends"])
    _, bounds = ref.attention(q, k, v, mask, None, do)
    g = gen(14)
    loss = lambda x: (ref.attention(*x, mask)[0][0] * do.double()).sum()
    x = [t.double() for t in (q, k, v)]
    for i in range(3):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = ([t + s * h * d if n == i else t for n, t in enumerate(x)] for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * h)
        bound = (bounds[i + 1] * d.abs()).sum() + 1e-6 * slope.abs()
        assert abs((got[i + 1].cpu().double() * d).sum() - slope) <= bound


def test_backward_is_deterministic_and_on_the_current_stream(device):
    q, k, v, do = _inputs(2, 300, 8, 2, 128, torch.bfloat16, seed=15)
    want = _run(device, q, k, v, do, window=100, sinks=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = _run(device, q, k, v, do, window=100, sinks=4)
    for a, b in zip(want, again):
        assert torch.equal(a, b)


def test_forward_in_a_graph(device):
    q, k, v, _ = (t.to(device) for t in _inputs(2, 130, 4, 2, 128, torch.bfloat16, seed=16))
    starts = torch.tensor([0, 9], dtype=torch.int32, device=device)
    with torch.no_grad():
        window_attention(q, k, v, window=50, sinks=1, starts=starts)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = window_attention(q, k, v, window=50, sinks=1, starts=starts)
        for i in range(3):
            q.copy_(torch.randn_like(q))
            starts.fill_(i)
            want = window_attention(q, k, v, window=50, sinks=1, starts=starts)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_no_tokens_and_no_gradient(device):
    q = torch.empty((2, 4, 0, 64), dtype=torch.bfloat16, device=device, requires_grad=True)
    out = window_attention(q, q[:, :2], q[:, :2])
    assert out.shape == q.shape
    out.sum().backward()
    q, k, v, _ = (t.to(device) for t in _inputs(1, 20, 2, 2, 64, torch.float16))
    assert not window_attention(q, k, v).requires_grad
    k.requires_grad_(True)
    window_attention(q, k, v).sum().backward()
    assert k.grad is not None and q.grad is None
