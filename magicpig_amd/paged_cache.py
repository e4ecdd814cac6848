"""`PagedKVCache` -- keys and values of many requests in pages, and the attention of each request's new tokens over them,
over the gfx950 C ABI (mp_paged_*).  What FlashInfer's append_paged_kv_cache and BatchDecodeWithPagedKVCacheWrapper are to
models/attnserver.py:73-106, 239-259, for one new token of a request or many (a chunk of its prompt, drafted tokens), with
rows as they come ("bf16") or quantised as they are written ("e4m3").

append, read and attention take the same description of their rows (int32 CUDA tensors):
    cu_seqlens [B + 1]   request b's new rows in the packed tensors: cu_seqlens[b] .. cu_seqlens[b + 1]
    page_table [B, P]    position p of request b lies in page page_table[b, p // page_size]
    kv_len     [B]       positions of request b, its new rows included
A request may have no new rows; rows outside every request, rows whose position would be below 0, and the rows of a request
whose kv_len its table cannot hold are not touched (check() reports the last).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from .prompt_attention import rows_strides, same_device, written


class PagedKVCache:
    def __init__(self):
        self._h = C.c_void_p()
        self._sizes = {}                       # workspace bytes by the sizes of a call
        L.check(L.lib().mp_paged_create(C.byref(self._h)))

    def __del__(self):
        try:
            if getattr(self, "_h", None) and self._h.value:
                L.lib().mp_paged_destroy(self._h)
                self._h = C.c_void_p()
        except Exception:
            pass

    def alloc(self, num_layers: int, num_attention_heads: int, num_key_value_heads: int, head_dim: int, num_pages: int,
              page_size: int = 64, kv_format: str = "bf16") -> None:
        """Pages of `page_size` tokens (a power of two up to 4096) for `num_layers` layers on the current device.
        kv_format "e4m3": a row -- one head's K or V of a token -- becomes e4m3 codes and one power of two, half the memory;
        an element then comes back off by at most 2^-4 of itself, or 2^-17 of its row's largest where that is more (magnitudes
        of 2^128 (1 - 2^-5) and more, the top of bf16's range, come back as infinities)."""
        if kv_format not in L.KV_FORMATS:
            raise ValueError(f"kv_format: expected one of {sorted(L.KV_FORMATS)}, got {kv_format!r}")
        L.check(L.lib().mp_paged_alloc(self._h, num_layers, num_attention_heads, num_key_value_heads, head_dim, num_pages,
                                       page_size, L.KV_FORMATS[kv_format]))
        self.num_layers, self.H, self.Hkv, self.D = num_layers, num_attention_heads, num_key_value_heads, head_dim
        self.num_pages, self.page_size, self.kv_format = num_pages, page_size, kv_format
        self._device = L.current_device()      # the handle's state lives here (the C ABI switches to it)

    def _rows(self, num_tokens, cu_seqlens, page_table, kv_len, **tensors):
        """Checks the description of a call's rows; returns its C arguments."""
        if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
            raise ValueError("page_table: expected a tensor [requests, pages]")
        B, P = page_table.shape
        L.expect(page_table, torch.int32, (B, P), "page_table")
        L.expect(cu_seqlens, torch.int32, (B + 1,), "cu_seqlens")
        L.expect(kv_len, torch.int32, (B,), "kv_len")
        same_device(self._device, cu_seqlens=cu_seqlens, page_table=page_table, kv_len=kv_len, **tensors)
        return cu_seqlens.data_ptr(), B, num_tokens, page_table.data_ptr(), P, kv_len.data_ptr()

    def append(self, layer_id: int, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, page_table: torch.Tensor,
               kv_len: torch.Tensor) -> None:
        """k, v bf16 [T, Hkv, D] (any token / head strides that are multiples of 8 elements) into the pages: row
        cu_seqlens[b] + i becomes position kv_len[b] - n_b + i of request b, n_b its number of new rows."""
        (T, kt, kh), (Tv, vt, vh) = rows_strides(k, self.Hkv, self.D, "k"), rows_strides(v, self.Hkv, self.D, "v")
        if T != Tv:
            raise ValueError(f"k, v: {T} and {Tv} tokens")
        rows = self._rows(T, cu_seqlens, page_table, kv_len, k=k, v=v)
        L.check(L.lib().mp_paged_append(self._h, layer_id, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, *rows,
                                        L.stream_on(self._device)))

    def read(self, layer_id: int, num_tokens: int, cu_seqlens: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor,
             k: torch.Tensor | None = None, v: torch.Tensor | None = None):
        """The rows append would write for this description, out of the pages: (k, v) bf16 [num_tokens, Hkv, D]."""
        shape = (num_tokens, self.Hkv, self.D)
        rows = self._rows(num_tokens, cu_seqlens, page_table, kv_len)
        if k is None:
            k = page_table.new_empty(shape, dtype=torch.bfloat16)
        if v is None:
            v = page_table.new_empty(shape, dtype=torch.bfloat16)
        written(k, torch.bfloat16, shape, "k")
        written(v, torch.bfloat16, shape, "v")
        same_device(self._device, k=k, v=v)
        L.check(L.lib().mp_paged_read(self._h, layer_id, k.data_ptr(), v.data_ptr(), *rows,
                                      L.stream_on(self._device)))
        return k, v

    def attention(self, layer_id: int, q: torch.Tensor, cu_seqlens: torch.Tensor, page_table: torch.Tensor,
                  kv_len: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None):
        """q bf16 [T, H, D]: row cu_seqlens[b] + i attends to positions 0 .. kv_len[b] - n_b + i of request b, as the pages hold
        them (append the rows' own keys first); query head h to kv head h // (H // Hkv).  Returns (out bf16 [T, H, D],
        lse f32 [T, H], base 2); a row that sees nothing gives 0 and -inf.  scale: default head_dim ** -0.5.  `out` may be q itself (any
        other overlap is refused).  Sums are f32, the
        weights are rounded to bf16 for the product with v."""
        H, D = self.H, self.D
        T, qt, qh = rows_strides(q, H, D, "q")
        if out is None:
            out = q.new_empty((T, H, D))
        else:
            written(out, torch.bfloat16, (T, H, D), "out")
        if lse is None:
            lse = q.new_empty((T, H), dtype=torch.float32)
        else:
            written(lse, torch.float32, (T, H), "lse")
        rows = self._rows(T, cu_seqlens, page_table, kv_len, q=q, out=out, lse=lse)
        size = self._workspace(rows[1], T, rows[4])
        # from torch's allocator: safe to reuse in stream order, and a captured graph's own
        work = q.new_empty((size,), dtype=torch.uint8) if size else None
        L.check(L.lib().mp_paged_attention(self._h, layer_id, q.data_ptr(), qt, qh, *rows, D ** -0.5 if scale is None else float(scale),
                                           out.data_ptr(), lse.data_ptr(), L.ptr(work), size,
                                           L.stream_on(self._device)))
        return out, lse

    def _workspace(self, requests: int, tokens: int, pages: int) -> int:
        """mp_paged_workspace: bytes, by the sizes alone."""
        key = (requests, tokens, pages)
        size = self._sizes.get(key)
        if size is None:
            need = C.c_int64()
            L.check(L.lib().mp_paged_workspace(self._h, requests, tokens, pages, C.byref(need)))
            if len(self._sizes) >= 4096:
                self._sizes.clear()
            size = self._sizes[key] = need.value
        return size

    def check(self) -> None:
        """Raise if a call since the last check met a page id or length outside the cache (waits for the current stream)."""
        L.check(L.lib().mp_paged_check(self._h, L.stream_on(self._device)))

    def get_pages(self, layer_id: int):
        """Views of the handle's memory: pages [num_pages, Hkv, page_size, 2 (K, V), D] in bf16 or float8_e4m3fn, and the rows'
        exponents + 127 u8 [num_pages, Hkv, page_size, 2] (None for "bf16")."""
        p, s = C.c_void_p(), C.c_void_p()
        L.check(L.lib().mp_paged_get_pages(self._h, layer_id, C.byref(p), C.byref(s)))
        shape, dev = (self.num_pages, self.Hkv, self.page_size, 2), torch.device("cuda", self._device)
        if self.kv_format == "bf16":
            return L.device_tensor(p.value, shape + (self.D,), "<i2", device=dev).view(torch.bfloat16), None
        return (L.device_tensor(p.value, shape + (self.D,), "|u1", device=dev).view(torch.float8_e4m3fn),
                L.device_tensor(s.value, shape, "|u1", device=dev))

    def footprint(self) -> dict:
        """HBM bytes per layer: rows and their exponents."""
        b = (C.c_int64 * 2)()
        L.check(L.lib().mp_paged_get_footprint(self._h, b))
        return {"pages": int(b[0]), "scales": int(b[1])}
