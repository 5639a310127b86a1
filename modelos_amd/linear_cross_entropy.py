"""Softmax cross entropy of a linear layer over a large vocabulary, without the logits in memory, on the HIP kernels.

`linear_cross_entropy(hidden, weight, labels)` is what a language model's head
and loss are together,

    F.cross_entropy((hidden @ weight.T).float(), labels)

in pieces of the vocabulary: the forward sums the exponentials of a piece's
logits and drops them, the backward computes them again, turns them into their
gradients and those into the piece's rows of weight's gradient and its part of
hidden's. The largest of it in memory are the gradients of one piece in 16 bits: up to
about 768 MB, and for more than 24576 tokens, whose pieces get no smaller than 16384
entries, 32 KB a token (2 GiB at 65536); beside them 4 bytes a number of hidden for its
gradient's sums and 2 for a scaled copy. The forward needs 8 bytes a token for every 128
entries. A training forward keeps a copy of the hidden states that count, and of a weight
that it had to copy for its rows (below), until its backward.

Tokens whose label is ignore_index, or lies outside [0, vocab), do not count:
their loss is 0, nothing is computed for them, what hidden holds there is not
used (it may be NaN) and their rows of its gradient are zeros. The mean is over
the tokens that count, and 0 if none does (where F.cross_entropy's is NaN). An infinite
weight makes its row's logits infinite or NaN; in the last 8 columns of a weight
whose rows are no multiple of 64 always NaN.

Logits, softmax sums and all other sums are float32, the loss is float32 and keeps
its precision down to 0. The gradients of the logits are rounded to the inputs'
type for the products they enter, in float16 in units of their token's own gradient,
so that gradients of any size, also of tokens far apart, keep their precision (in
weight's gradient, which sums over tokens, those whose product with the hidden state
is no smaller than 2^-29 of the call's largest); up to 128 tokens they enter
as two such numbers, and what the rounding leaves of the label's is made up for in hidden's
gradient. Sums run in a fixed order: losses and gradients are bitwise
deterministic.

Supported: bfloat16 and float16, up to 65536 numbers a row,
fewer than 2^22 tokens and 2^30 entries, on the GPU; anything else raises NotImplementedError.
Under torch.autocast hidden and weight are cast to its type first, as a linear layer's
are, and get gradients of their own type (a float32 table is cast in every call).
There is no CPU path: CPU tensors raise. The backward cannot be differentiated
again, and there are no forward-mode derivatives: dual tensors raise
NotImplementedError.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _lib
from .embedding_bag import _require_device
from .window_attention import _refuse_tangents

_DTYPES = (torch.bfloat16, torch.float16)
_CAST = (*_DTYPES, torch.float32)  # what autocast casts
_LABELS = {torch.int32: 32, torch.int64: 64}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_MAX_TOKENS, _MAX_VOCAB, _MAX_DIM, _MAX_STRIDE = 1 << 22, 1 << 30, 65536, 1 << 22


def _buffer(n: int, device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


def _readable(weight: torch.Tensor) -> torch.Tensor:
    """weight itself if the kernels can read its rows, in whole vectors of 16 bytes, else a copy with longer rows."""
    V, D = weight.shape
    if D % 8 == 0 and weight.stride(1) == 1 and weight.stride(0) % 8 == 0 and D <= weight.stride(0) <= _MAX_STRIDE \
            and weight.data_ptr() % 16 == 0:
        return weight
    return F.pad(weight, (0, -D % 8)).contiguous() if D % 8 else weight.clone(memory_format=torch.contiguous_format)


def _forward(x, weight, dim: int, labels, ignore: int, reduction: int):
    n, V, dev = x.shape[0], weight.shape[0], x.device
    lib = _lib.load()
    loss = torch.empty(labels.shape if reduction == 0 else (), dtype=torch.float32, device=dev)
    kept = _buffer(lib.pkm_linear_ce_kept_size(n, dim), dev)
    ws = _buffer(lib.pkm_linear_ce_fwd_workspace_size(n, V, dim), dev)
    _lib.call_on(dev, "pkm_linear_ce_fwd", _lib.ptr(x), x.stride(0), n, _lib.ptr(weight), weight.stride(0), V, dim,
                 _lib.dtype_code(x), _lib.ptr(labels), _LABELS[labels.dtype], ignore, reduction, _lib.ptr(loss), _lib.ptr(kept),
                 kept.numel(), _lib.ptr(ws), ws.numel(), _lib.stream_of(dev))
    return loss, kept


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore: int, reduction: int):
        dim = hidden.shape[-1]
        readable = _readable(weight)
        loss, kept = _forward(_rows(hidden), readable, dim, labels, ignore, reduction)
        ctx.save_for_backward(kept, readable)
        ctx.rest = (hidden.shape, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        kept, weight = ctx.saved_tensors
        shape, reduction = ctx.rest
        dim, V, dev = shape[-1], weight.shape[0], weight.device
        n = shape.numel() // dim
        grad_loss = grad_loss.contiguous()
        dx = torch.empty(shape, dtype=weight.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty((V, dim), dtype=weight.dtype, device=dev) if ctx.needs_input_grad[1] else None
        ws = _buffer(_lib.load().pkm_linear_ce_bwd_workspace_size(n, V, dim), dev)
        _lib.call_on(dev, "pkm_linear_ce_bwd", _lib.ptr(kept), kept.numel(), n, _lib.ptr(weight), weight.stride(0), V, dim,
                     _lib.dtype_code(weight), _lib.ptr(grad_loss), reduction, _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(ws),
                     ws.numel(), _lib.stream_of(dev))
        return dx, dw, None, None, None


def _rows(hidden: torch.Tensor) -> torch.Tensor:
    """hidden as [tokens, dim] with contiguous rows."""
    x = hidden.reshape(-1, hidden.shape[-1])
    return x if x.stride(1) == 1 and x.stride(0) >= 0 else x.contiguous()


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of hidden @ weight.T against labels.

    hidden: [..., dim]; weight: [vocab, dim] of hidden's type; labels: int32 or int64 of hidden's shape without the last.
    ignore_index: the label of tokens that do not count. reduction: "mean" over the tokens that count, "sum", or "none"
    (a loss for each label). Any strides; rows of weight that are not whole, aligned 16-byte vectors (a dim that is no
    multiple of 8 among them) cost a copy of it in every call.
    Returns float32.
    """
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear_cross_entropy: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} are not "
                         "[..., dim] and [vocab, dim]")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: labels {tuple(labels.shape)} do not match hidden {tuple(hidden.shape)}")
    if labels.dtype not in _LABELS:
        raise TypeError(f"linear_cross_entropy: labels must be int32 or int64, got {labels.dtype}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction {reduction!r} has to be 'mean', 'sum' or 'none'")
    if not isinstance(ignore_index, int) or isinstance(ignore_index, bool) or not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"linear_cross_entropy: ignore_index {ignore_index!r} has to be a whole number of 64 bits")
    if torch.is_autocast_enabled("cuda"):  # as F.linear there
        dtype = torch.get_autocast_dtype("cuda")
        hidden, weight = (t.to(dtype) if t.is_cuda and t.dtype in _CAST else t for t in (hidden, weight))
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise NotImplementedError(f"linear_cross_entropy: {hidden.dtype} with a weight of {weight.dtype} is not supported "
                                  "(bfloat16 and float16 are, both alike)")
    if labels.numel() >= _MAX_TOKENS or weight.shape[1] > _MAX_DIM or weight.shape[0] >= _MAX_VOCAB:
        raise NotImplementedError(f"linear_cross_entropy: {labels.numel()} tokens, a weight of {tuple(weight.shape)} are not "
                                  f"supported (fewer than {_MAX_TOKENS} tokens, rows of up to {_MAX_DIM} numbers are)")
    _refuse_tangents("linear_cross_entropy", hidden, weight)
    _require_device(hidden, weight, labels)
    labels, code = labels.contiguous(), _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropyFn.apply(hidden, weight, labels, ignore_index, code)
    return _forward(_rows(hidden), _readable(weight), weight.shape[1], labels, ignore_index, code)[0]


__all__ = ["linear_cross_entropy"]
