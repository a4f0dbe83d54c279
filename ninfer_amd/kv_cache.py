"""KV cache planes for one attention layer (reference src/core/kv_cache.{h,cpp}).

Layout per layer (reference plan_kv_cache, src/core/kv_cache.cpp:55-99): codes I8 [D, P, Hkv]
and FP16 scales [D/64, P, Hkv] for K and for V, or BF16 values [D, P, Hkv] and no scales, with
P = align_up(max_context, 128). A trailing batch dimension B stacks independent sequences (one
contiguous region per sequence).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _capi
from ._capi import KVLayerView, PagedBlockView, PagedKVLayerView, Tensor
from .device import DeviceArray

QUANT_GROUP = 64


def align_up(v: int, a: int) -> int:
    return (v + a - 1) // a * a


class KVCacheLayer:
    """Owning cache planes (INT8-G64 by default, or BF16) and the matching nmi_kv_layer_view."""

    def __init__(self, max_context: int, num_kv_heads: int, head_dim: int, batch: int = 1,
                 dtype: int = _capi.I8):
        if max_context <= 0 or max_context > 0x7FFFFFFF:
            raise ValueError("KVCache max_context out of range")
        if num_kv_heads <= 0 or head_dim <= 0 or head_dim % QUANT_GROUP:
            raise ValueError("KVCache geometry invalid")
        if dtype not in (_capi.I8, _capi.BF16):
            raise ValueError("KVCache dtype must be I8 or BF16")
        self.dtype = dtype
        self.max_context = max_context
        self.padded_context = align_up(max_context, 128)
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.batch = batch
        P = self.padded_context
        G = head_dim // QUANT_GROUP
        self.k = DeviceArray(dtype, (head_dim, P, num_kv_heads, batch))
        self.v = DeviceArray(dtype, (head_dim, P, num_kv_heads, batch))
        if dtype == _capi.I8:
            self.k_scale = DeviceArray(_capi.FP16, (G, P, num_kv_heads, batch))
            self.v_scale = DeviceArray(_capi.FP16, (G, P, num_kv_heads, batch))
        else:
            self.k_scale = self.v_scale = None

    def _planes(self):
        return [a for a in (self.k, self.v, self.k_scale, self.v_scale) if a is not None]

    def zero(self, stream=None) -> None:
        for a in self._planes():
            a.zero(stream)

    def view(self) -> KVLayerView:
        v = KVLayerView()
        v.k = self.k.tensor()
        v.v = self.v.tensor()
        if self.k_scale is not None:
            v.k_scale = self.k_scale.tensor()
            v.v_scale = self.v_scale.tensor()
        v.max_context = self.max_context
        v.padded_context = self.padded_context
        v.num_kv_heads = self.num_kv_heads
        v.head_dim = self.head_dim
        v.dtype = self.dtype
        v.quant_group = QUANT_GROUP if self.dtype == _capi.I8 else 0
        return v

    def payload_bytes(self) -> int:
        return sum(a.nbytes for a in self._planes())

    # host views in the reference's order: codes[b][h][pos][d], scales[b][h][pos][g]
    # (BF16: (k, v) values[b][h][pos][d])
    def download(self):
        P, H, D, B = self.padded_context, self.num_kv_heads, self.head_dim, self.batch
        if self.dtype == _capi.BF16:
            return (self.k.numpy().reshape(B, H, P, D), self.v.numpy().reshape(B, H, P, D))
        G = D // QUANT_GROUP
        return (
            self.k.numpy().reshape(B, H, P, D),
            self.v.numpy().reshape(B, H, P, D),
            self.k_scale.numpy().reshape(B, H, P, G),
            self.v_scale.numpy().reshape(B, H, P, G),
        )

    def upload(self, k_codes, v_codes, k_scales=None, v_scales=None) -> None:
        self.k.upload(k_codes)
        self.v.upload(v_codes)
        if self.k_scale is not None:
            self.k_scale.upload(k_scales)
            self.v_scale.upload(v_scales)


class PagedKVCacheLayer:
    """Owning pool of pages (INT8-G64 by default, or BF16), the table of `batch` sequences of up to `max_pages` pages
    (-1: absent, as at first), the counts of the table's entries per page (`refs`) and the matching nmi_paged_kv_layer_view.
    `block_size`: means of blocks of so many keys next to the pages (0: none). `table_of`: the layer whose table and counts this one
    shares, as the layers of a model do."""

    def __init__(self, pages: int, page_size: int, num_kv_heads: int, head_dim: int, batch: int, max_pages: int, dtype: int = _capi.I8,
                 block_size: int = 0, table_of: "PagedKVCacheLayer | None" = None):
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError("PagedKVCache page_size must be a power of two in [16, 4096]")
        if pages <= 0 or batch <= 0 or max_pages <= 0:
            raise ValueError("PagedKVCache capacity must be positive")
        if num_kv_heads <= 0 or head_dim <= 0 or head_dim % QUANT_GROUP:
            raise ValueError("PagedKVCache geometry invalid")
        if dtype not in (_capi.I8, _capi.BF16):
            raise ValueError("PagedKVCache dtype must be I8 or BF16")
        if block_size and (block_size < 32 or block_size > page_size or block_size & (block_size - 1)):
            raise ValueError("PagedKVCache block_size must be a power of two from 32 to page_size")
        if table_of is not None and (table_of.pages, table_of.page_size, table_of.batch, table_of.max_pages) != (pages, page_size, batch, max_pages):
            raise ValueError("PagedKVCache layers that share a table must have the same pages")
        self.pages, self.page_size, self.num_kv_heads, self.head_dim = pages, page_size, num_kv_heads, head_dim
        self.batch, self.max_pages, self.dtype = batch, max_pages, dtype
        self.k = DeviceArray(dtype, (head_dim, page_size, num_kv_heads, pages))
        self.v = DeviceArray(dtype, (head_dim, page_size, num_kv_heads, pages))
        self.k_scale = self.v_scale = None
        if dtype == _capi.I8:
            self.k_scale = DeviceArray(_capi.FP16, (head_dim // QUANT_GROUP, page_size, num_kv_heads, pages))
            self.v_scale = DeviceArray(_capi.FP16, (head_dim // QUANT_GROUP, page_size, num_kv_heads, pages))
        self.block_size = block_size
        self.block_codes = self.block_scales = None
        if block_size:
            self.block_codes = DeviceArray(_capi.I8, (head_dim, page_size // block_size, num_kv_heads, pages))
            self.block_scales = DeviceArray(_capi.FP32, (page_size // block_size, num_kv_heads, pages))
        if table_of is not None:
            self.page_table, self.refs = table_of.page_table, table_of.refs
        else:
            self.page_table = DeviceArray(_capi.I32, (max_pages, batch))
            self.refs = DeviceArray(_capi.I32, (pages,))
            self.set_pages(np.full((batch, max_pages), -1, dtype=np.int32))

    def _planes(self):
        return [a for a in (self.k, self.v, self.k_scale, self.v_scale) if a is not None]

    def zero(self, stream=None) -> None:
        for a in self._planes():
            a.zero(stream)

    def set_pages(self, table) -> None:
        """The whole page table, int32 [batch, max_pages], and the counts that belong to it."""
        table = np.asarray(table, dtype=np.int32).reshape(self.batch, self.max_pages)
        self.page_table.upload(table)
        held = table[(table >= 0) & (table < self.pages)]
        self.refs.upload(np.bincount(held, minlength=self.pages).astype(np.int32))

    def blocks(self) -> PagedBlockView:
        v = PagedBlockView()
        if self.block_codes is None:
            raise ValueError("this cache keeps no block means")
        v.codes, v.scales, v.block_size = self.block_codes.tensor(), self.block_scales.tensor(), self.block_size
        return v

    def view(self) -> PagedKVLayerView:
        v = PagedKVLayerView()
        v.k, v.v = self.k.tensor(), self.v.tensor()
        if self.k_scale is not None:
            v.k_scale, v.v_scale = self.k_scale.tensor(), self.v_scale.tensor()
        v.page_table = self.page_table.tensor()
        v.page_size, v.num_kv_heads, v.head_dim = self.page_size, self.num_kv_heads, self.head_dim
        v.dtype = self.dtype
        v.quant_group = QUANT_GROUP if self.dtype == _capi.I8 else 0
        return v

    # host views: planes [page][h][row][d], scales [page][h][row][g]
    def download(self):
        N, H, R, D = self.pages, self.num_kv_heads, self.page_size, self.head_dim
        return tuple(a.numpy().reshape(N, H, R, n) for a, n in zip(self._planes(), (D, D, D // QUANT_GROUP, D // QUANT_GROUP)))

    def upload(self, *planes) -> None:
        for a, x in zip(self._planes(), planes, strict=True):
            a.upload(x)
