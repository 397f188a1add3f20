"""A paged key/value cache in 8 bits.

``QuantCache`` holds keys and values of ``num_pages`` pages of ``page_size`` slots, every head of a
slot as 8-bit levels with one float32 scale: amax = max |x| of the head, scale = amax / top, level =
round(x * (top / amax)), top 127 ("int8") or 448 ("e4m3").  Rows are quantised as they are written
and widened as they are read back; who owns which page is the caller's business (slots and page
tables are plain index tensors, as everywhere in ``ops``).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import Q8_FORMATS, check, dtype_code, lib, stream_ptr

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_I64x2 = ctypes.c_int64 * 2


class QuantCache:
    """``k`` / ``v``: [num_pages, page_size, num_heads, head_dim] levels (int8 or float8_e4m3fn);
    ``k_scale`` / ``v_scale``: float32 [num_pages, page_size, num_heads].  A slot is page *
    page_size + offset.  A fresh cache reads as zeros."""

    def __init__(self, num_pages: int, page_size: int, num_heads: int, head_dim: int, fmt: str = "int8", device="cuda"):
        if fmt not in Q8_FORMATS:
            raise ValueError(f"QuantCache: fmt must be one of {sorted(Q8_FORMATS)}")
        if min(num_pages, page_size, num_heads, head_dim) < 1:
            raise ValueError("QuantCache: sizes must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("QuantCache requires a CUDA device")
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.num_heads, self.head_dim, self.fmt = int(num_heads), int(head_dim), fmt
        self._code, store = Q8_FORMATS[fmt]
        shape = (self.num_pages, self.page_size, self.num_heads)
        self.k = torch.zeros(shape + (self.head_dim,), dtype=torch.int8, device=device).view(store)
        self.v = torch.zeros(shape + (self.head_dim,), dtype=torch.int8, device=device).view(store)
        self.k_scale = torch.zeros(shape, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(shape, dtype=torch.float32, device=device)
        # where the writers of one slot settle which token keeps it; zero between calls
        self._owner = torch.zeros((self.num_slots,), dtype=torch.int32, device=device)

    @property
    def num_slots(self) -> int:
        return self.num_pages * self.page_size

    @property
    def device(self):
        return self.k.device

    def _status(self, what: str, status):
        if status is None:
            return None
        self._on_device(what, status.buf)
        return status.ptr

    def _on_device(self, what: str, *ts: torch.Tensor) -> None:
        device = self.k.get_device()
        for t in ts:
            if t.get_device() != device:
                if not t.is_cuda:
                    raise RuntimeError(f"{what} requires CUDA tensors")
                raise ValueError(f"{what}: operand on {t.device}, the cache is on {self.device}")

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, status=None) -> None:
        """Token i of k and v ([tokens, num_heads, head_dim], float32 / float16 / bfloat16, any
        strides) goes to slot ``slots[i]`` (int64 or int32).  A negative slot skips the token
        (padding); a slot behind the cache is skipped and counted in ``status`` (an
        ops.IndexStatus, checked against ``num_slots``) when one is given.  Of several tokens with
        one slot the last is kept.  Writes to one slot from two streams must be ordered by the
        caller."""
        what = "QuantCache.write"
        self._on_device(what, k, v, slots)
        if k.dtype not in _FLOATS or v.dtype != k.dtype:
            raise TypeError(f"{what}: k and v must be float32, float16 or bfloat16 of one dtype")
        if slots.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{what}: slots must be int64 or int32")
        if slots.dim() != 1:
            raise ValueError(f"{what}: slots must be 1-D")
        want = (slots.shape[0], self.num_heads, self.head_dim)
        if tuple(k.shape) != want or tuple(v.shape) != want:
            raise ValueError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)}, expected {want}")
        if slots.shape[0] == 0:
            return
        if k.stride(-1) != 1 and self.head_dim > 1:
            k = k.contiguous()
        if v.stride(-1) != 1 and self.head_dim > 1:
            v = v.contiguous()
        slots = slots.contiguous()
        check(lib().vbt_b200_kv_cache_write(
            self.k.data_ptr(), self.k_scale.data_ptr(), self.v.data_ptr(), self.v_scale.data_ptr(), self.num_slots,
            self.num_heads, self.head_dim, self._code, k.data_ptr(), _I64x2(*k.stride()[:2]), v.data_ptr(),
            _I64x2(*v.stride()[:2]), dtype_code(k.dtype), slots.data_ptr(), dtype_code(slots.dtype), slots.shape[0],
            self._owner.data_ptr(), self._status(what, status), stream_ptr(self.k)))

    def read(self, page_table: torch.Tensor, starts: torch.Tensor, total: Optional[int] = None,
             dtype: torch.dtype = torch.bfloat16, out=None, status=None):
        """The sequences' keys and values, one behind the other: rows starts[s] .. starts[s + 1) of
        the results hold sequence s, whose position p lies in page ``page_table[s, p // page_size]``.

        page_table: int64 or int32 [sequences, pages]; starts: int64 [sequences + 1], ascending, on the
        device.  Returns (k, v), each [total, num_heads, head_dim] of ``dtype``; rows that no
        sequence owns are zero.  With ``out`` (a pair of dense tensors) their row count and dtype
        count instead of ``total`` and ``dtype``, and rows that no sequence owns are left as they
        are.  A page outside the cache, a position behind the table's last page, or one in front of
        its sequence (starts that do not ascend) reads as zeros and is counted in ``status`` (an
        ops.IndexStatus, checked against ``num_pages``) when one is given."""
        what = "QuantCache.read"
        self._on_device(what, page_table, starts)
        if page_table.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{what}: page_table must be int64 or int32")
        if starts.dtype != torch.int64:
            raise TypeError(f"{what}: starts must be int64")
        if page_table.dim() != 2 or starts.dim() != 1 or starts.shape[0] != page_table.shape[0] + 1:
            raise ValueError(f"{what}: page_table must be [sequences, pages] and starts [sequences + 1]")
        if out is None:
            if total is None or total < 0:
                raise ValueError(f"{what}: total, the number of rows, is needed without out")
            if dtype not in _FLOATS:
                raise TypeError(f"{what} gives float32, float16 or bfloat16")
            ko = self.k.new_empty(int(total), self.num_heads, self.head_dim, dtype=dtype)
            vo = torch.empty_like(ko)
        else:
            ko, vo = out
            self._on_device(what, ko, vo)
            if ko.dtype not in _FLOATS or vo.dtype != ko.dtype:
                raise TypeError(f"{what}: out must be float32, float16 or bfloat16 of one dtype")
            if ko.dim() != 3 or tuple(ko.shape[1:]) != (self.num_heads, self.head_dim) or ko.shape != vo.shape or \
                    not ko.is_contiguous() or not vo.is_contiguous():
                raise ValueError(f"{what}: out must be two dense [rows, {self.num_heads}, {self.head_dim}] tensors")
            if ko.numel() and abs(ko.data_ptr() - vo.data_ptr()) < ko.numel() * ko.element_size():
                raise ValueError(f"{what}: the two outputs overlap")
        if ko.shape[0] == 0:
            return ko, vo
        if page_table.stride(-1) != 1 and page_table.shape[1] > 1:
            page_table = page_table.contiguous()
        starts = starts.contiguous()
        check(lib().vbt_b200_kv_cache_read(
            ko.data_ptr(), vo.data_ptr(), dtype_code(ko.dtype), ko.shape[0], self.k.data_ptr(), self.k_scale.data_ptr(),
            self.v.data_ptr(), self.v_scale.data_ptr(), self.num_slots, self.page_size, self.num_heads, self.head_dim,
            self._code, page_table.data_ptr() if page_table.numel() else None, dtype_code(page_table.dtype), page_table.stride(0),
            page_table.shape[1], starts.data_ptr(), page_table.shape[0], int(out is None),
            self._status(what, status), stream_ptr(self.k)))
        return ko, vo
