"""A paged key / value cache in 4 bits on the HIP kernels, and attention over it.

`Int4KVCache` holds the keys and values of one layer's decoded tokens:
`append` quantises new ones into their pages, `read` gives them back in 16
bits, `attend` answers a few query tokens per sequence from it.

A head vector is held in groups of 32 numbers: minimum m and step
s = (max - min) / 15 in the cache's type, codes c = round((x - m) / s); the
number read back is m + s c, within s / 2 of x up to the rounding of m, s and
the result. Numbers have to be finite, and far enough from the type's ends that
max - min and m + 15 s stay inside it; attend needs steps of 0 or between 2^-100 and 2^100. With the parameters a number takes 5
bits instead of 16.

Pages are the caller's to hand out: `table` [batch, width] (int32, on the
device) names each sequence's pages, position t lies in page
table[b, t // page_size]. Positions outside the table and entries that are no
page are left out: not written, read as zeros, not visible. Every call runs on
the current stream, reads lengths and tables on the device and does not
synchronise, so it can be captured into a graph.

Supported: bfloat16 and float16, head dims 64 and 128, pages of a multiple of
16 tokens, on the GPU; anything else raises NotImplementedError.
"""
from __future__ import annotations

import torch

from . import _lib
from .embedding_bag import _require_device
from .window_attention import _DIMS, _DTYPES, _check_scale, _check_window, _refuse_tangents

GROUP = 32
_MAX_POSITIONS = 1 << 30  # of a sequence's table; the entry point takes fewer


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [batch, heads, tokens, dim] itself if the kernels can read its strides, else a copy."""
    sb, sh, st, sd = t.stride()
    fits = sd == 1 and t.data_ptr() % 16 == 0 and (sb | sh | st) % 8 == 0
    return t if fits else t.clone(memory_format=torch.contiguous_format)


class Int4KVCache:
    """Keys and values of one layer in 4-bit codes, in pages.

    codes: uint8 [2 (K, V), pages, kv_heads, page_size, dim / 2];
    params: dtype [2 (K, V), pages, kv_heads, 2 (s, m), dim / 32, page_size].
    Number d = w + 16 i (w < 16) of a vector lies in its word w; dim 128: 32-bit
    words, bits 4 (i // 2 + 4 (i % 2)); dim 64: 16-bit words, bits 4 i.
    """

    def __init__(self, pages: int, kv_heads: int, dim: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, n in (("pages", pages), ("kv_heads", kv_heads), ("page_size", page_size)):
            if not isinstance(n, int) or isinstance(n, bool) or n < 1:
                raise ValueError(f"Int4KVCache: {name} {n!r} has to be a whole number of at least 1")
        if dim not in _DIMS or dtype not in _DTYPES or page_size % 16 != 0 or page_size > 4096:
            raise NotImplementedError(f"Int4KVCache: heads of {dim} in {dtype}, pages of {page_size} are not supported "
                                      "(64 or 128 in bfloat16 or float16, multiples of 16 up to 4096 are)")
        self.pages, self.kv_heads, self.dim, self.page_size = pages, kv_heads, dim, page_size
        self.codes = torch.zeros((2, pages, kv_heads, page_size, dim // 2), dtype=torch.uint8, device=device)
        self.params = torch.zeros((2, pages, kv_heads, 2, dim // GROUP, page_size), dtype=dtype, device=device)

    @property
    def dtype(self) -> torch.dtype:
        return self.params.dtype

    @property
    def device(self) -> torch.device:
        return self.params.device

    def __repr__(self):
        return (f"Int4KVCache(pages={self.pages}, kv_heads={self.kv_heads}, dim={self.dim}, "
                f"page_size={self.page_size}, dtype={self.dtype}, device={self.device})")

    def _sizes(self):
        return (_lib.ptr(self.codes), _lib.ptr(self.params), self.pages, self.kv_heads, self.page_size, self.dim,
                _lib.dtype_code(self.params))

    def _check_plan(self, what: str, batch: int, table: torch.Tensor, **counts: torch.Tensor):
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != batch:
            raise ValueError(f"{what}: table has to be int32 [{batch}, width], got {table.dtype} {tuple(table.shape)}")
        for name, t in counts.items():
            if t.dtype != torch.int32 or t.shape != (batch,):
                raise ValueError(f"{what}: {name} has to be int32 [{batch}], got {t.dtype} {tuple(t.shape)}")
        _require_device(self.params, table, *counts.values())

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
               counts: torch.Tensor) -> None:
        """Writes k, v [batch, kv_heads, tokens, dim]: token t < counts[b] of sequence b becomes position
        starts[b] + t (starts, counts: int32 [batch] on the device)."""
        if k.dim() != 4 or k.shape != v.shape or k.shape[1] != self.kv_heads or k.shape[3] != self.dim:
            raise ValueError(f"Int4KVCache.append: k {tuple(k.shape)}, v {tuple(v.shape)} are not "
                             f"[batch, {self.kv_heads}, tokens, {self.dim}]")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise ValueError(f"Int4KVCache.append: k and v have to be {self.dtype}, got {k.dtype} and {v.dtype}")
        B, _, T, _ = k.shape
        self._check_plan("Int4KVCache.append", B, table, starts=starts, counts=counts)
        _require_device(self.params, k, v)
        k, v, table, starts, counts = _rows(k), _rows(v), table.contiguous(), starts.contiguous(), counts.contiguous()
        _lib.call_on(self.device, "pkm_kv4_append", *self._sizes(), _lib.heads(k), _lib.heads(v), _lib.ptr(table),
                     table.shape[1], _lib.ptr(starts), _lib.ptr(counts), B, T, _lib.stream_of(self.device))

    def read(self, table: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor,
             tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """k, v [batch, kv_heads, tokens, dim] of positions starts[b] + t; zeros for t >= counts[b]."""
        if not isinstance(tokens, int) or isinstance(tokens, bool) or tokens < 0:
            raise ValueError(f"Int4KVCache.read: tokens {tokens!r} has to be a whole number of at least 0")
        B = table.shape[0]
        self._check_plan("Int4KVCache.read", B, table, starts=starts, counts=counts)
        table, starts, counts = table.contiguous(), starts.contiguous(), counts.contiguous()
        k, v = (torch.empty((B, self.kv_heads, tokens, self.dim), dtype=self.dtype, device=self.device)
                for _ in range(2))
        _lib.call_on(self.device, "pkm_kv4_read", *self._sizes(), _lib.ptr(table), table.shape[1], _lib.ptr(starts),
                     _lib.ptr(counts), B, tokens, _lib.heads(k), _lib.heads(v), _lib.stream_of(self.device))
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, window: int | None = None,
               sinks: int = 0, scale: float | None = None) -> torch.Tensor:
        """Attention of q [batch, q_heads, queries, dim], each sequence's last tokens, over what the cache holds.

        lengths: int32 [batch] on the device, tokens of each sequence, the queries' own (already appended)
        among them. Query i stands at p = lengths[b] - queries + i and sees the positions j <= p with
        p - j < window or j < sinks (window None: all). Returns [batch, q_heads, queries, dim]; rows that
        see nothing are zeros. There are no derivatives: q that requires a gradient or has a tangent is refused.
        """
        if q.dim() != 4 or q.shape[3] != self.dim or q.shape[1] == 0 or q.shape[1] % self.kv_heads != 0:
            raise ValueError(f"Int4KVCache.attend: q {tuple(q.shape)} is not [batch, q_heads, queries, {self.dim}] "
                             f"with q_heads a multiple of {self.kv_heads}")
        if q.dtype != self.dtype:
            raise ValueError(f"Int4KVCache.attend: q has to be {self.dtype}, got {q.dtype}")
        if torch.is_grad_enabled() and q.requires_grad:
            raise RuntimeError("Int4KVCache.attend has no backward; call it under torch.no_grad() or detach q")
        _refuse_tangents("Int4KVCache.attend", q)
        window, sinks = _check_window(window, sinks, _MAX_POSITIONS)
        scale = _check_scale(scale, self.dim)
        B, H, Q, D = q.shape
        self._check_plan("Int4KVCache.attend", B, table, lengths=lengths)
        _require_device(self.params, q)
        q, table, lengths = _rows(q), table.contiguous(), lengths.contiguous()
        width = table.shape[1]
        out = torch.empty((B, H, Q, D), dtype=q.dtype, device=q.device)
        ws_bytes = _lib.load().pkm_kv4_attend_workspace_size(B, H, self.kv_heads, Q, D, width, self.page_size, window,
                                                            sinks)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        _lib.call_on(self.device, "pkm_kv4_attend", *self._sizes(), _lib.heads(q), _lib.ptr(table), width,
                     _lib.ptr(lengths), B, H, Q, window, sinks, scale, _lib.heads(out), _lib.ptr(ws), ws_bytes,
                     _lib.stream_of(self.device))
        return out
