"""The paged key/value cache of include/wsp_hip.h (wsp_hip_paged_*): the pool's
tensors and the rows of a call, which KernelContext.paged_append, paged_read and
paged_attention take.

    cache = PagedCache.allocate("E4M3", pages=512, heads=20, page_rows=32, head_width=64)
    rows = PagedRows(starts, lengths, table, rows=n, max_count=1, max_length=448)
    context.paged_append(cache, rows, keys, values)
    context.paged_attention(cache, rows, q, heads=20, causal=True, scale=0.125, out=out)

Which sequence owns which page is the caller's to keep: a row of the table names
a sequence's pages in the order of its positions. starts, lengths and the table
stay on the device and are read when the kernels run, so a captured graph
follows what they hold at each replay (up to the max_length it was captured
with).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _native as N
from .decoder import LogicError

STORAGES = {"F32": (N.WSP_F32, torch.float32), "F16": (N.WSP_F16, torch.float16),
            "BF16": (N.WSP_BF16, torch.bfloat16), "E4M3": (N.WSP_E4M3, torch.float8_e4m3fn)}
_CODES = {dtype: code for code, dtype in STORAGES.values()}


_FLOAT = torch.float32
_MOST = 2 ** 31 - 1  # of an extent


class PagedCache:
    """A pool over tensors keys and values [pages, heads, page_rows, head_width]
    in fp32, fp16, bf16 or float8_e4m3fn; the last has exponent bytes [pages,
    heads, page_rows] for each (a row's values are its E4M3 values times
    2^(byte - 127)). Holds on to the tensors; their contents are theirs."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_exponents: Optional[torch.Tensor] = None,
                 value_exponents: Optional[torch.Tensor] = None):
        if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != values.dtype:
            raise ValueError("keys and values are pools [pages, heads, page_rows, head_width] of one type")
        if keys.dtype not in _CODES:
            raise LogicError(f"a paged cache holds fp32, fp16, bf16 or float8_e4m3fn, and not {keys.dtype}")
        exponents = [t for t in (key_exponents, value_exponents) if t is not None]
        if len(exponents) != (2 if keys.dtype == torch.float8_e4m3fn else 0):
            raise ValueError("float8_e4m3fn pools, and no others, have exponents for keys and for values")
        if any(t.shape != keys.shape[:3] or t.dtype != torch.uint8 for t in exponents):
            raise ValueError("exponents are bytes [pages, heads, page_rows]")
        self._keep = [keys, values] + exponents
        if not all(t.is_contiguous() for t in self._keep):
            raise ValueError("the pool's tensors are contiguous")
        if len({t.device for t in self._keep}) != 1:
            raise ValueError("the pool's tensors lie on one device")
        self.keys, self.values, self.key_exponents, self.value_exponents = keys, values, key_exponents, value_exponents
        self.pages, self.heads, self.page_rows, self.head_width = keys.shape
        self.width = self.heads * self.head_width  # of a packed row
        self.device = keys.get_device()  # -1: not a GPU's
        self._ctable = N.wsp_paged_cache(_CODES[keys.dtype], self.pages, self.page_rows, self.heads, self.head_width,
                                         keys.data_ptr(), values.data_ptr(),
                                         *(t.data_ptr() for t in exponents or ()))
        self.table = ctypes.byref(self._ctable)

    @classmethod
    def allocate(cls, storage: str, pages: int, heads: int, page_rows: int, head_width: int,
                 device: int = 0) -> "PagedCache":
        """A pool of its own, its slots not set (nothing reads a slot before it
        is written)."""
        if storage not in STORAGES:
            raise LogicError(f"a paged cache holds {', '.join(STORAGES)}, and not {storage}")
        shape = (pages, heads, page_rows, head_width)
        pools = [torch.empty(shape, dtype=STORAGES[storage][1], device=f"cuda:{device}") for _ in range(2)]
        exponents = [torch.empty(shape[:3], dtype=torch.uint8, device=f"cuda:{device}")
                     for _ in range(2 if storage == "E4M3" else 0)]
        return cls(*pools, *exponents)


class PagedRows:
    """The packed rows of a call and their sequences (wsp_paged_rows): starts
    [sequences + 1], lengths [sequences] (the new rows among them) and the table
    [sequences, table_width] of page ids, int32; `rows` the packed tensors' rows,
    max_count and max_length bounds on a sequence's new rows and its length."""

    def __init__(self, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, rows: int, max_count: int,
                 max_length: int):
        self._keep = (starts, lengths, table)
        if any(t.dtype != torch.int32 or not t.is_contiguous() for t in self._keep):
            raise ValueError("starts, lengths and the table are contiguous int32 tensors")
        sequences = lengths.numel()
        if starts.dim() != 1 or lengths.dim() != 1 or starts.numel() != sequences + 1 or table.dim() != 2 \
                or table.shape[0] != sequences:
            raise ValueError("starts is [sequences + 1], lengths [sequences] and the table [sequences, table_width]")
        if len({t.device for t in self._keep}) != 1:
            raise ValueError("starts, lengths and the table lie on one device")
        if not all(0 <= n <= _MOST for n in (rows, max_count, max_length, table.shape[1])):
            raise ValueError(f"{rows} rows, at most {max_count} of {max_length} positions a sequence")
        self.rows = rows
        self.device = lengths.get_device()
        self._ctable = N.wsp_paged_rows(sequences, rows, max_count, max_length, table.shape[1], starts.data_ptr(),
                                        lengths.data_ptr(), table.data_ptr())
        self.table = ctypes.byref(self._ctable)

    def check(self, cache: PagedCache, device: int) -> None:
        if cache.device != device or self.device != device:
            raise ValueError(f"a pool on device {cache.device} and rows on {self.device} for a context on device {device}")

    def stride(self, tensor: torch.Tensor, width: int, device: int) -> int:
        """How far the packed rows of `tensor` lie apart."""
        shape, strides = tensor.shape, tensor.stride()
        if tensor.dtype is not _FLOAT or len(shape) != 2 or shape[0] < self.rows or shape[1] != width or strides[1] != 1:
            raise ValueError(f"packed rows are fp32 [{self.rows}, {width}], each row in one run")
        if tensor.get_device() != device:
            raise ValueError(f"a tensor on {tensor.device} for a context on device {device}")
        apart = strides[0] if shape[0] > 1 else width
        if apart > _MOST:
            raise ValueError(f"packed rows {apart} floats apart (at most {_MOST})")
        return apart
