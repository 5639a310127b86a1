"""Cross entropy of a linear layer: arguments that are refused, on the CPU before any kernel runs."""
from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from modelos_amd.linear_cross_entropy import linear_cross_entropy

P = ctypes.c_void_p(1 << 20)
BF16 = torch.bfloat16
X, W, Y = torch.zeros(3, 8, dtype=BF16), torch.zeros(5, 8, dtype=BF16), torch.zeros(3, dtype=torch.long)


@pytest.fixture(scope="module")
def lib():
    from modelos_amd import _lib, build_lib

    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    return _lib.load()


@pytest.mark.parametrize("x,w,y,options,error", [
    (X, W[:, :7], Y, {}, ValueError), (X, W[0], Y, {}, ValueError), (X[:, :0], W[:, :0], Y, {}, ValueError),
    (X, W[:0], Y, {}, ValueError), (X, W, Y[:2], {}, ValueError), (X, W, Y[:, None], {}, ValueError),
    (X[0, 0], W, Y[0], {}, ValueError), (X, W, Y.short(), {}, TypeError), (X, W, Y.float(), {}, TypeError),
    (X, W, Y, {"reduction": "max"}, ValueError), (X, W, Y, {"ignore_index": 1.0}, ValueError),
    (X, W, Y, {"ignore_index": True}, ValueError), (X, W, Y, {"ignore_index": 1 << 63}, ValueError),
    (X.float(), W.float(), Y, {}, NotImplementedError), (X, W.half(), Y, {}, NotImplementedError),
    (X[:1].expand(1 << 22, 8), W, Y[:1].expand(1 << 22), {}, NotImplementedError),
    (X[:, :1].expand(3, 65537), W[:, :1].expand(5, 65537), Y, {}, NotImplementedError),
    (X, W, Y, {}, RuntimeError),  # CPU tensors
])
def test_refused(x, w, y, options, error):
    with pytest.raises(error):
        linear_cross_entropy(x, w, y, **options)


@pytest.mark.parametrize("dual", [0, 1])
def test_dual_tensors_are_refused(dual):
    t = [X, W]
    with forward_ad.dual_level():
        t[dual] = forward_ad.make_dual(t[dual], torch.ones_like(t[dual]))
        with pytest.raises(NotImplementedError, match="forward"):
            linear_cross_entropy(*t, Y)


def _forward(lib, x=P, x_stride=64, tokens=10, w=P, w_stride=64, vocab=100, dim=64, dtype=1, labels=P, bits=64, reduction=1, loss=P,
             kept=P, kept_bytes=1 << 62, ws=P, ws_bytes=1 << 62):
    return lib.pkm_linear_ce_fwd(x, x_stride, tokens, w, w_stride, vocab, dim, dtype, labels, bits, -100, reduction, loss, kept,
                                 kept_bytes, ws, ws_bytes, None)


def _backward(lib, tokens=10, w=P, w_stride=64, vocab=100, dim=64, dtype=1, grad=P, reduction=1, dx=P, dw=P, kept=P,
              kept_bytes=1 << 62, ws=P, ws_bytes=1 << 62):
    return lib.pkm_linear_ce_bwd(kept, kept_bytes, tokens, w, w_stride, vocab, dim, dtype, grad, reduction, dx, dw, ws, ws_bytes,
                                 None)


ODD = ctypes.c_void_p((1 << 20) + 8)
COMMON = [
    (dict(tokens=-1), 1), (dict(vocab=0), 1), (dict(dim=0), 1), (dict(dtype=0), 2), (dict(dtype=9), 2), (dict(tokens=1 << 22), 2),
    (dict(dim=65537), 2), (dict(vocab=1 << 30), 2), (dict(vocab=(1 << 30) - 1, tokens=1 << 16), 2), (dict(reduction=3), 1),
    (dict(w=None), 1), (dict(w=ODD), 1), (dict(w_stride=63), 1), (dict(w_stride=68), 1), (dict(dim=65, w_stride=64), 1),
    (dict(w_stride=1 << 23), 1), (dict(kept=None), 3), (dict(kept=ODD), 3), (dict(kept_bytes=255), 3), (dict(ws=None), 3),
    (dict(ws=ODD), 3), (dict(ws_bytes=255), 3),
]


@pytest.mark.parametrize("args,status", COMMON + [
    (dict(x=None), 1), (dict(labels=None), 1), (dict(loss=None), 1), (dict(bits=16), 1), (dict(x_stride=-1), 1)])
def test_entry_forward(lib, args, status):
    assert _forward(lib, **args) == status


@pytest.mark.parametrize("args,status", COMMON + [(dict(grad=None), 1), (dict(dx=ODD), 1), (dict(dw=ODD), 1)])
def test_entry_backward(lib, args, status):
    assert _backward(lib, **args) == status


def test_sizes(lib):
    assert lib.pkm_linear_ce_kept_size(1 << 22, 64) == lib.pkm_linear_ce_kept_size(10, 0) == 0
    assert lib.pkm_linear_ce_fwd_workspace_size(10, 0, 64) == lib.pkm_linear_ce_bwd_workspace_size(10, 1 << 30, 64) == 0
    # 16384 tokens, 151936 entries: no more than 768 MB of the logits' gradients at a time, and 67 MB of dx's sums
    assert 16384 * 16384 < lib.pkm_linear_ce_bwd_workspace_size(16384, 151936, 1024) < (768 << 20) + 70e6


@pytest.mark.parametrize("dim", [64, 1000, 4096])
@pytest.mark.parametrize("vocab", [300, 151936])
@pytest.mark.parametrize("tokens", [100, 16384, 24576, 65536, 1 << 18, 1 << 20])
def test_sizes_of_long_batches(lib, tokens, vocab, dim):
    """What the documentation says a call needs: one piece's gradients, 768 MB or 32 KB a token, hidden's sums and copy; sums of
    128 entries each in the forward. Tokens and widths count in whole tiles of 256, widths of a copy in 64; the sums of few
    tokens are split, up to 256 tiles."""
    up = lambda n, to: -(-n // to) * to
    n, few = up(tokens, 256), 256 * 256 * 256 * 4
    pieces = min(max(768 << 20, 32768 * n), 2 * n * up(vocab, 256))
    rest = n * (4 * up(dim, 256) + 2 * up(dim, 64) + 16) + 256
    split = 256 * 256 * 256 * 4 if vocab == 300 else 0  # dW's sums, where the vocabulary is one piece
    assert lib.pkm_linear_ce_bwd_workspace_size(tokens, vocab, dim) <= pieces + rest + few + split
    assert lib.pkm_linear_ce_fwd_workspace_size(tokens, vocab, dim) <= n * (8 * up(vocab, 256) // 128 + 1) + 4096
