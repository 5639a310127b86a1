"""Token embedding with a scale, and the gradient of its table by sorted tokens, on the HIP kernels.

`token_embedding(ids, weight, scale=, padding_idx=)` is what a decoder reads its
tokens with:

    out[..., :] = scale * weight[ids[...], :]

in one pass, rounded once to weight's type. The gradient of the table is dense
(every row is written; rows without a token are zeros) and summed in float32 in
the order of the tokens, so it is bitwise deterministic, however often a token
occurs. The row of padding_idx is read as any other and gets no gradient. Ids
outside [0, rows) read zeros and give no gradient.

`TokenEmbedding` is the module: the parameter `weight` as nn.Embedding has it.

Supported: float32, bfloat16 and float16 tables, int32 and int64 ids, rows of
any length (those of whole, aligned 16-byte vectors are read and written so), on
the GPU. There is no CPU path: CPU tensors raise. The backward cannot be
differentiated again, and there are no forward-mode derivatives: dual tensors
raise NotImplementedError.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib
from .embedding_bag import _require_device
from .window_attention import _refuse_tangents

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_IDS = {torch.int32: 32, torch.int64: 64}
_MAX = 1 << 31  # tokens, rows


def _forward(ids, weight, scale: float):
    rows, dim = weight.shape
    out = torch.empty((*ids.shape, dim), dtype=weight.dtype, device=weight.device)
    _lib.call_on(weight.device, "pkm_embed_fwd", _lib.ptr(ids), _IDS[ids.dtype], ids.numel(), _lib.ptr(weight), rows,
                 weight.stride(0), dim, _lib.dtype_code(weight), scale, _lib.ptr(out), _lib.stream_of(weight.device))
    return out


class _TokenEmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale: float, padding: int):
        ctx.save_for_backward(ids)
        ctx.rest = (weight.shape, scale, padding)
        return _forward(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        (rows, dim), scale, padding = ctx.rest
        grad_out = grad_out.contiguous()
        dw = torch.empty((rows, dim), dtype=grad_out.dtype, device=grad_out.device)
        ws_bytes = _lib.load().pkm_embed_bwd_workspace_size(ids.numel(), rows, dim)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dw.device)
        _lib.call_on(dw.device, "pkm_embed_bwd", _lib.ptr(ids), _IDS[ids.dtype], ids.numel(), _lib.ptr(grad_out), rows, dim,
                     _lib.dtype_code(dw), padding, scale, _lib.ptr(dw), _lib.ptr(ws), ws_bytes,
                     _lib.stream_of(dw.device))
        return None, dw, None, None


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                    padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[ids], [*ids.shape, dim] of weight's type.

    ids: int32 or int64 of any shape and strides. weight: [rows, dim]; rows may lie
    apart. padding_idx: a row in [-rows, rows) that gets no gradient.
    """
    if weight.dim() != 2 or weight.shape[1] == 0:
        raise ValueError(f"token_embedding: weight {tuple(weight.shape)} is not [rows, dim]")
    if ids.dtype not in _IDS:
        raise TypeError(f"token_embedding: ids must be int32 or int64, got {ids.dtype}")
    rows, dim = weight.shape
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"token_embedding: scale {scale!r} has to be finite")
    padding = -1
    if padding_idx is not None:
        if not isinstance(padding_idx, int) or isinstance(padding_idx, bool) or not -rows <= padding_idx < rows:
            raise ValueError(f"token_embedding: padding_idx {padding_idx!r} is not a row of {rows}")
        padding = padding_idx % rows
    if weight.dtype not in _DTYPES:
        raise NotImplementedError(f"token_embedding: a table of {weight.dtype} is not supported "
                                  "(float32, bfloat16 and float16 are)")
    if ids.numel() >= _MAX or rows >= _MAX or dim >= 1 << 24:
        raise NotImplementedError(f"token_embedding: {ids.numel()} tokens, a table of {tuple(weight.shape)} are not "
                                  "supported (fewer than 2^31 tokens and rows, 2^24 numbers a row are)")
    _refuse_tangents("token_embedding", weight)
    _require_device(ids, weight)
    ids = ids.contiguous()
    if weight.stride(1) != 1 or not dim <= weight.stride(0) < _MAX:
        weight = weight.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _TokenEmbeddingFn.apply(ids, weight, scale, padding)
    return _forward(ids, weight, scale)


class TokenEmbedding(nn.Module):
    """nn.Embedding (its parameter `weight` and its initialisation) on token_embedding, with a scale."""

    def __init__(self, rows: int, dim: int, padding_idx: int | None = None, *, scale: float = 1.0, device=None, dtype=None):
        super().__init__()
        self.padding_idx, self.scale = padding_idx, scale
        self.weight = nn.Parameter(torch.empty((rows, dim), device=device, dtype=dtype))
        nn.init.normal_(self.weight)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return token_embedding(ids, self.weight, scale=self.scale, padding_idx=self.padding_idx)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, {self.weight.shape[1]}, padding_idx={self.padding_idx}, scale={self.scale}"


__all__ = ["token_embedding", "TokenEmbedding"]
