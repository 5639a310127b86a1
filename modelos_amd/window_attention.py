"""Causal attention through a sliding window with first tokens that stay visible, on the HIP kernels.

`window_attention(q, k, v, window=, sinks=, starts=, ends=)` is the attention
of a decoder layer over a (padded) batch, forward and backward. Key j is
visible to the query at position p of a sequence of tokens [start, end) if

    start <= j <= p < end  and  (p - j < window  or  j - start < sinks)

and out_p = sum_j softmax_j(scale q_p.k_j) v_j over the visible keys. Rows that
see no key, those of padding among them, are zeros in the output and in the
gradients; what the inputs hold there is not used (it may be NaN). Key heads
are shared by consecutive groups of query heads; their gradients are summed
over the group in a fixed order, so the backward is deterministic. A row that
sees one key alone has the weight 1 whatever q and k are: its gradients to both
are exactly 0.

Logits, softmax statistics and sums are float32. The softmax weights, and in
the backward their gradients, are rounded to the inputs' type for the matrix
products they enter, as the inputs are; in float16 with a power of two taken out
of the gradients, so that any size of grad_out keeps its precision.

Supported: bfloat16 and float16, head dims 64 and 128, on the GPU; anything
else raises NotImplementedError. There is no CPU path: CPU tensors raise.
The backward cannot be differentiated again, and there are no forward-mode
derivatives: dual tensors raise NotImplementedError.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .embedding_bag import _require_device

_DTYPES = (torch.bfloat16, torch.float16)
_DIMS = (64, 128)
_MAX_TOKEN_STRIDE = 1 << 22  # elements; tiles are addressed with 32-bit offsets
_MAX_TOKENS = 1 << 24
# Training keeps what the rounding of the output left for the backward's <grad_out, out>, for all rows up to this window and
# else for so many first rows of each sequence (PKM_ATTN_REST_TOKENS). The fewer keys a row sees, the more of its gradient an error
# there is: without it the error of dq is 2.4 times that of a mere rounding of dq at 2 keys, 1.5 times at 20 and 1.35 at 200
# (with it 1.1 to 1.2); for all rows at a window of 1024, where it is 1.3, keeping it would cost 1 to 6 % of a training step
# (4 x 4096 tokens, 16 / 8 heads of 128).
_REST_TOKENS = 256


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t [batch, heads, tokens, dim] itself if the kernels can read its strides, else a copy."""
    B, H, T, D = t.shape
    sb, sh, st, sd = t.stride()
    fits = sd == 1 and (T <= 1 or D <= st) and st < _MAX_TOKEN_STRIDE and t.data_ptr() % 16 == 0
    return t if fits and (sb | sh | st) % 8 == 0 else t.clone(memory_format=torch.contiguous_format)


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor of t's shape, its tokens outside its heads if t's are (a projection's layout)."""
    B, H, T, D = t.shape
    if t.stride(1) < t.stride(2):
        return torch.empty((B, T, H, D), dtype=t.dtype, device=t.device).transpose(1, 2)
    return torch.empty((B, H, T, D), dtype=t.dtype, device=t.device)


def _bound(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.contiguous()


def _forward(q, k, v, starts, ends, window: int, sinks: int, scale: float, rest, lse):
    B, H, T, D = q.shape
    out = _empty_like(q)
    _lib.call_on(q.device, "pkm_window_attn_fwd", _lib.heads(q), _lib.heads(k), _lib.heads(v), _lib.ptr(starts),
                 _lib.ptr(ends), B, H, k.shape[1], T, D, _lib.dtype_code(q), window, sinks, scale, _lib.heads(out),
                 _lib.heads(rest), _lib.ptr(lse), _lib.stream_of(q.device))
    return out


class _WindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, ends, window: int, sinks: int, scale: float):
        q, k, v = _readable(q), _readable(k), _readable(v)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
        B, H, T, D = q.shape
        kept = T if 0 < window <= _REST_TOKENS else min(T, _REST_TOKENS)
        rest = torch.empty((B, H, kept, D), dtype=q.dtype, device=q.device)
        out = _forward(q, k, v, starts, ends, window, sinks, scale, rest, lse)
        ctx.save_for_backward(q, k, v, out, rest, lse, starts, ends)
        ctx.sizes = (window, sinks, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, rest, lse, starts, ends = ctx.saved_tensors
        B, H, T, D = q.shape
        grad_out = _readable(grad_out)
        dq, dk, dv = _empty_like(q), _empty_like(k), _empty_like(v)
        ws_bytes = _lib.load().pkm_window_attn_bwd_workspace_size(B, H, k.shape[1], T, D, *ctx.sizes[:2])
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=q.device)
        _lib.call_on(q.device, "pkm_window_attn_bwd", _lib.heads(q), _lib.heads(k), _lib.heads(v), _lib.heads(out),
                     _lib.heads(rest), _lib.ptr(lse), _lib.heads(grad_out), _lib.ptr(starts), _lib.ptr(ends), B, H, k.shape[1], T, D,
                     _lib.dtype_code(q), *ctx.sizes, _lib.heads(dq), _lib.heads(dk), _lib.heads(dv), _lib.ptr(ws),
                     ws_bytes, _lib.stream_of(q.device))
        return dq, dk, dv, None, None, None, None, None


def _check_window(window, sinks, most: int) -> tuple[int, int]:
    """window (0: none) and sinks, cut to `most`, which no sequence reaches: the entry points take 64-bit sizes."""
    if window is not None and (not isinstance(window, int) or isinstance(window, bool) or window < 1):
        raise ValueError(f"window {window!r} has to be a whole number of at least 1, or None")
    if not isinstance(sinks, int) or isinstance(sinks, bool) or sinks < 0:
        raise ValueError(f"sinks {sinks!r} has to be a whole number of at least 0")
    return min(window or 0, most), min(sinks, most)


def _check_scale(scale, dim: int) -> float:
    scale = dim**-0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale {scale!r} has to be positive and finite")
    return scale


def _refuse_tangents(what: str, *tensors: torch.Tensor) -> None:
    """The kernels read the primal numbers alone: a dual tensor's tangent would be lost."""
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                     starts: torch.Tensor | None = None, ends: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention of q [B, q_heads, T, dim] over k, v [B, kv_heads, T, dim].

    window: keys a query sees behind it, itself among them (None: all).
    sinks: first tokens of each sequence that every later query sees.
    starts, ends: int32 [B] on the device, each sequence's first token and the
    one behind its last (default: 0 and T; clamped to [0, T]).
    scale: of the logits, positive (default: dim ** -0.5).
    Any strides; those with contiguous heads, 16-byte aligned, are read in place.
    Returns [B, q_heads, T, dim] of q's type, laid out as q.
    """
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"window_attention: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} are not "
                         "q [B, q_heads, T, dim] and k, v [B, kv_heads, T, dim]")
    B, H, T, D = q.shape
    if k.shape[0] != B or k.shape[2] != T or k.shape[3] != D or k.shape[1] == 0 or H == 0 or H % k.shape[1] != 0:
        raise ValueError(f"window_attention: q {tuple(q.shape)} does not match k {tuple(k.shape)} "
                         "(the same batch, tokens and dim, kv_heads dividing q_heads)")
    window, sinks = _check_window(window, sinks, _MAX_TOKENS)
    scale = _check_scale(scale, D)
    for name, t in (("starts", starts), ("ends", ends)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (B,)):
            raise ValueError(f"window_attention: {name} has to be int32 [{B}], got {t.dtype} {tuple(t.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype or D not in _DIMS:
        raise NotImplementedError(f"window_attention: heads of {D} in {q.dtype} / {k.dtype} / {v.dtype} are not "
                                  "supported (64 or 128 in bfloat16 or float16 are)")
    if T >= _MAX_TOKENS:
        raise NotImplementedError(f"window_attention: {T} tokens are not supported (fewer than {_MAX_TOKENS} are)")
    _refuse_tangents("window_attention", q, k, v)
    _require_device(q, k, v, *(t for t in (starts, ends) if t is not None))
    starts, ends = _bound(starts), _bound(ends)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttentionFn.apply(q, k, v, starts, ends, window, sinks, scale)
    return _forward(_readable(q), _readable(k), _readable(v), starts, ends, window, sinks, scale, None, None)
