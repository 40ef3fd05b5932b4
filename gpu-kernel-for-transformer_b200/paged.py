"""The paged KV cache: its pool of pages and the batches that use it.

``PagedKVCache`` holds keys and values of many sequences of different lengths
in pages, in fp16 or in 8 bits with a scale per token and head;
``PagedBatch`` says which tokens of which sequences a step deals with.
``ops.paged_append``, ``ops.paged_read`` and ``ops.paged_attention`` take the
two. (The contiguous cache of ``UserOptimizedTransformer.enable_kv_cache``, the
reference's torch_transformer_benchmark.py:409-462, keeps sequences of one
length and fp16 only.)

Both hold tensors and the C structure that describes them, built once; neither
reads device memory, so both can be made and used while a graph is captured.
Which page a token lives on is the caller's to decide (``page_table``): there is
no allocator here.
"""

from __future__ import annotations

import ctypes
import itertools
from typing import Optional

import torch

from . import _lib

_CODES = {
    torch.float16: _lib.TFX_CACHE_F16,
    torch.int8: _lib.TFX_CACHE_INT8,
    torch.float8_e4m3fn: _lib.TFX_CACHE_E4M3,
}


_INT_MAX = 2 ** 31 - 1  # sizes are ints in the C structures, and ctypes cuts what is longer


_GEOMETRIES: dict = {}  # sizes that decide an attention call's workspace -> a small number
_NUMBERS = itertools.count()  # (len() of the table could give two threads the same one)


class _Fixed:
    """Attributes that the C structure (`_ref`, set last) was built from: not to be replaced."""

    def __setattr__(self, name, value):
        if "_ref" in self.__dict__:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed once the object is made: "
                                 "write into its tensors, or make another")
        super().__setattr__(name, value)


class PagedKVCache(_Fixed):
    """A pool of ``num_pages`` pages of ``page_size`` tokens (16, 32, 64, 128 or 256).

    ``dtype``: ``torch.float16``; or ``torch.int8`` / ``torch.float8_e4m3fn``,
    with an fp32 scale for each token and head (``head_dim`` 16 and up):
    a cached value is code * scale. ``head_dim``: 8, 16, 32, 64, 128 or 256.

    ``k``, ``v``: [num_pages, page_size, kv_heads, head_dim] views;
    ``k_scale``, ``v_scale``: [num_pages, kv_heads, page_size], or None.
    In memory a page holds its tokens head by head (each head's part of a page
    is one block); ``from_tensors`` takes any other order. The pool is not
    cleared: a token is read only where a batch's ``kv_len`` counts it.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device="cuda") -> None:
        shape = (num_pages, kv_heads, page_size, head_dim)
        scales = (None, None)
        if dtype != torch.float16:
            scales = tuple(torch.empty(shape[:3], dtype=torch.float32, device=device)
                           for _ in range(2))
        self._bind(torch.empty(shape, dtype=dtype, device=device).transpose(1, 2),
                   torch.empty(shape, dtype=dtype, device=device).transpose(1, 2), *scales)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor,
                     k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """A cache over the caller's tensors, which it keeps and writes in place.

        ``k``, ``v``: [num_pages, page_size, kv_heads, head_dim], the same
        strides, the last dimension contiguous and the others multiples of 16
        bytes; scales [num_pages, kv_heads, page_size] fp32, contiguous.
        """
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        if k.dtype not in _CODES:
            raise ValueError(f"cache dtype must be float16, int8 or float8_e4m3fn, got {k.dtype}")
        if k.ndim != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(
                "k and v must be [num_pages, page_size, kv_heads, head_dim] of one dtype and device")
        pages, page_size, heads, hd = k.shape
        strides = _strides(k)
        if strides != _strides(v) or strides[3] != 1:
            raise ValueError("k and v must have the same strides, the last dimension contiguous")
        if max(pages, page_size, heads) > _INT_MAX:
            raise ValueError("num_pages, page_size and kv_heads must be below 2^31")
        quant = k.dtype != torch.float16
        for s in (k_scale, v_scale):
            if (s is not None) != quant:
                raise ValueError("8-bit caches need k_scale and v_scale, fp16 ones take none")
            if quant and (s.shape != (pages, heads, page_size) or s.dtype != torch.float32
                          or not s.is_contiguous() or s.device != k.device):
                raise ValueError("scales must be contiguous float32 [num_pages, kv_heads, page_size]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.dtype, self.device = k.dtype, k.device
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, heads, hd
        self._struct = _lib.TfxPagedCache(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if quant else None,
            v_scale.data_ptr() if quant else None, _CODES[k.dtype], pages, page_size, heads, hd,
            *strides[:3])
        self._half = k.new_empty(0, dtype=torch.float16)  # outputs are allocated from it
        self._index = k.device.index if k.device.type == "cuda" else None
        self._scale = hd ** -0.5
        self._geometry = _GEOMETRIES.setdefault((heads, hd, page_size, k.dtype), next(_NUMBERS))
        self._ref = ctypes.byref(self._struct)


def _strides(t: torch.Tensor):
    """Strides, those of dimensions of size 1 (which address nothing) as if contiguous."""
    out, at = list(t.stride()), 1
    for d in range(t.ndim - 1, -1, -1):
        if t.shape[d] == 1:
            out[d] = max(at, t.shape[-1]) if d < t.ndim - 1 else 1
        at = max(at, out[d] * t.shape[d])
    return tuple(out)


class PagedBatch(_Fixed):
    """The sequences of one step, their new tokens packed one behind the other.

    ``page_table`` int32 [B, max_pages]: the pages of each sequence in order of
    position (an id outside the pool: no page; its keys are masked, writes to
    it dropped); ``query_start`` int32 [B + 1]: sequence b owns rows
    query_start[b] .. query_start[b+1] - 1 of the packed tensors; ``kv_len`` int32
    [B]: its tokens in all, the new ones included, which are the last of them.
    ``num_tokens``: rows of the packed tensors; rows behind query_start[B]
    belong to no sequence and are left as they are.

    ``max_query_len`` (default ``num_tokens``): no sequence has more new tokens;
    attention leaves further ones out. ``max_kv_len`` (default: what the page
    table can hold): a bound on ``kv_len``, which only decides how the keys are
    split over the GPU.

    The device tensors are kept and read when a kernel runs, so a captured
    graph sees what they hold at its replay. (Write into them; attributes cannot
    be replaced.)
    """

    def __init__(self, page_table: torch.Tensor, query_start: torch.Tensor, kv_len: torch.Tensor,
                 num_tokens: int, max_query_len: Optional[int] = None,
                 max_kv_len: Optional[int] = None) -> None:
        if page_table.ndim != 2 or page_table.shape[0] < 1 or page_table.shape[1] < 1:
            raise ValueError("page_table must be [B, max_pages]")
        b, width = page_table.shape
        if query_start.shape != (b + 1,) or kv_len.shape != (b,):
            raise ValueError("query_start must be [B + 1] and kv_len [B]")
        for t in (page_table, query_start, kv_len):
            if t.dtype != torch.int32:
                raise ValueError("page_table, query_start and kv_len must be int32")
            if t.device != page_table.device:
                raise ValueError("page_table, query_start and kv_len must be on one device")
        if width > 1 and page_table.stride(1) != 1 or not query_start.is_contiguous() or \
                not kv_len.is_contiguous():
            raise ValueError("rows of page_table, query_start and kv_len must be contiguous")
        if num_tokens < 0 or (max_query_len or 0) < 0 or (max_kv_len or 0) < 0:
            raise ValueError("num_tokens, max_query_len and max_kv_len must not be negative")
        if max(b, width, num_tokens) > _INT_MAX:
            raise ValueError("B, max_pages and num_tokens must be below 2^31")
        self.page_table, self.query_start, self.kv_len = page_table, query_start, kv_len
        self.device, self.num_tokens = page_table.device, num_tokens
        self._index = page_table.device.index if page_table.device.type == "cuda" else None
        self.max_query_len = num_tokens if max_query_len is None else max_query_len
        self.max_kv_len = (1 << 30) if max_kv_len is None else max_kv_len
        self._struct = _lib.TfxPagedBatch(
            page_table.data_ptr(), page_table.stride(0) if b > 1 else width, width,
            query_start.data_ptr(), kv_len.data_ptr(), b, num_tokens, min(self.max_query_len, num_tokens),
            min(self.max_kv_len, 1 << 30))
        self._workspaces = {}
        self._ref = ctypes.byref(self._struct)

    def _workspace_bytes(self, lib, cache: PagedKVCache, q_heads: int) -> int:
        """Workspace of an attention call (a function of sizes only, looked up once)."""
        key = q_heads << 32 | cache._geometry
        need = self._workspaces.get(key)
        if need is None:
            with torch.cuda.device(self._index):  # the plan follows the device's SM count
                need = lib.tfx_paged_attention_workspace_bytes(cache._ref, self._ref, q_heads)
            self._workspaces[key] = need
        return need
