"""A paged key/value cache held in 4 bits, for single-token decoding.

DenseCore keeps no cache (its SDPA, python/densecore/functional.py:276, takes whole keys and
values); :class:`KVCache4` stands beside the float32 decode of
:func:`densecore_b200.functional.scaled_dot_product_attention` and holds a context in 5 bits a value.
"""
from __future__ import annotations

import numbers

import torch
from torch.autograd import forward_ad

from . import _lib, _native


def _whole(name, value, least):
    if type(value) is not int and (isinstance(value, bool) or not isinstance(value, numbers.Integral)):
        raise TypeError(f"{name} must be a whole number")
    if value < least:
        raise ValueError(f"{name} must be at least {least}")
    if value >= 1 << 62:
        raise ValueError(f"{name} is out of range")
    return int(value)


def _counts(name, t, batch=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a Tensor")
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if batch is not None and tuple(t.shape) != (batch,):
        raise ValueError(f"{name} must be ({batch},), got {tuple(t.shape)}")


class KVCache4:
    """``num_pages`` pages of ``page_size`` tokens of ``kv_heads`` heads of ``head_dim`` channels.

    Position p of sequence b lies in slot ``p % page_size`` of page ``page_table[b, p // page_size]``.
    The caller owns page tables (B, P), lengths and positions (B), all int32 tensors on the cache's
    device, and hands out pages; sequences may share pages that none of them appends to. Each group of
    32 channels of a token is held as low (its least value, rounded down to bfloat16), scale (a
    fifteenth of its range, rounded up to bfloat16) and 4-bit codes, and stands for
    low + scale * code: within half a scale of the value, about 3 % of the group's range. A group with
    an infinity or a NaN reads as NaN.

    The contents of tables and lengths are checked on the device: an entry out of range is not
    written, reads as zero or is left out of the attention, lengths are clamped to the table, and
    ``dc_device_status`` reports 3. Calls are asynchronous on the current stream; an append and a read of the
    same pages belong on one stream or need an event between them.
    """

    def __init__(self, num_pages, kv_heads, head_dim, page_size=64, device="cuda"):
        num_pages, kv_heads = _whole("num_pages", num_pages, 1), _whole("kv_heads", kv_heads, 1)
        page_size = _whole("page_size", page_size, 16)
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page_size % 16:
            raise ValueError("page_size must be a multiple of 16")
        self.num_pages, self.kv_heads, self.head_dim, self.page_size = num_pages, kv_heads, int(head_dim), page_size
        self._hold(torch.zeros((num_pages, kv_heads, page_size // 16, 20 * self.head_dim), dtype=torch.uint8, device=device))

    def _hold(self, data):
        self._data, self.device = data, data.device
        self._desc = _lib.DcCache4(data.data_ptr(), self.num_pages, self.kv_heads, self.head_dim, self.page_size)

    @property
    def data(self):
        """The pages, uint8 (num_pages, kv_heads, page_size / 16, 20 head_dim). A page is contiguous: copying
        one is copying ``data[page]``; a whole cache is restored with ``data.copy_()``."""
        return self._data

    def __getstate__(self):
        return {name: value for name, value in self.__dict__.items() if name != "_desc"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._hold(self._data)

    def _table(self, page_table):
        _counts("page_table", page_table)
        if page_table.dim() != 2:
            raise ValueError("page_table must be (B, pages)")
        if page_table.device != self.device:
            raise RuntimeError(f"the page table is on {page_table.device}, the cache on {self.device}")
        return page_table.shape[0]

    def _eager(self):
        """The pages are no tensors of a trace, which would keep nothing of a call."""
        if _native._traced("a 4-bit cache"):
            raise RuntimeError("a 4-bit cache cannot be traced")

    def append(self, key, value, page_table, start, end=None):
        """Token i of key, value (B, kv_heads, T, head_dim) to position ``start[b] + i``, where that is
        below ``end[b]`` (ragged prompts). Places from ``end`` on keep what they hold. One call must
        not write a slot twice. Keys and values are taken detached: no gradient or tangent passes the cache."""
        self._eager()
        b = self._table(page_table)
        _counts("start", start, b)
        if end is not None:
            _counts("end", end, b)
        for name, t in (("key", key), ("value", value)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"cache {name} must be a Tensor")
            if t.dtype not in (torch.float32, torch.float16, torch.bfloat16) or t.dtype != key.dtype:
                raise TypeError("cache key and value must both be float32, float16 or bfloat16")
            if t.dim() != 4 or t.shape[0] != b or t.shape[1] != self.kv_heads or t.shape[3] != self.head_dim:
                raise ValueError(f"cache {name} must be ({b}, {self.kv_heads}, T, {self.head_dim}), got {tuple(t.shape)}")
        if key.shape != value.shape:
            raise ValueError("cache key and value must have one shape")
        _native._cache4_append(self._desc, key.detach(), value.detach(), page_table, start, end)

    def read(self, page_table, lengths, max_length):
        """(key, value) of the first ``max_length`` positions in float32, (B, kv_heads, max_length,
        head_dim), zeros from ``lengths[b]`` on."""
        self._eager()
        b = self._table(page_table)
        _counts("lengths", lengths, b)
        return _native._cache4_read(self._desc, page_table, lengths, _whole("max_length", max_length, 0))

    def attention(self, query, page_table, lengths, scale=None, window=None, sinks=0, return_lse=False):
        """softmax(query @ key^T * scale) @ value of one token per sequence, (B, H, 1, head_dim) in
        float32, float16 or bfloat16, over its first ``lengths[b]`` positions; H a multiple of
        kv_heads (grouped queries). With ``window`` the token, standing at the last position, sees the
        positions less than ``window`` back and the first ``sinks``. scale defaults to
        1/sqrt(head_dim). An empty sequence gives 0. No gradient.

        The softmax's weights keep 24 bits for float32 queries and 16 for the others; a query keeps 28 bits
        below its largest channel, or 22 where several heads share a key head. Scores and sums are held in
        32 bits. :func:`densecore_b200.set_sdpa_precision` does not apply."""
        self._eager()
        b = self._table(page_table)
        _counts("lengths", lengths, b)
        if not isinstance(query, torch.Tensor):
            raise TypeError("cache attention query must be a Tensor")
        if query.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise TypeError(f"cache attention query must be float32, float16 or bfloat16, got {query.dtype}")
        if query.dim() != 4 or query.shape[0] != b or query.shape[2] != 1 or query.shape[3] != self.head_dim:
            raise ValueError(f"cache attention query must be ({b}, H, 1, {self.head_dim}), got {tuple(query.shape)}")
        if query.shape[1] % self.kv_heads:
            raise ValueError(f"query heads must be a multiple of the cache's {self.kv_heads}")
        if (query.requires_grad and torch.is_grad_enabled()
                or forward_ad._current_level >= 0 and forward_ad.unpack_dual(query).tangent is not None):
            raise NotImplementedError("attention over a 4-bit cache has no gradient")
        if scale is not None and (isinstance(scale, bool) or not isinstance(scale, numbers.Real)):
            raise TypeError("scale must be real")
        window = 0 if window is None else _whole("window", window, 1)
        out, lse = _native._cache4_attention(self._desc, query, page_table, lengths, window,
                                             _whole("sinks", sinks, 0), scale, return_lse)
        return (out, lse) if return_lse else out
