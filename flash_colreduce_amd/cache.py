"""A paged cache of keys and values, quantised or not: what a caller that prunes by `flash_colreduce` keeps, and what its next
tokens attend to.

    cache = KVCache.zeros(pages, heads, page_size, head_dim, torch.int8)
    cache_write(cache, key, value, table, start)                     # (B, H, T, D) to positions start ..
    k, v = cache_read(cache, table, lengths, n)                      # (B, H, n, D), for flash_colreduce
    keep = topk_keep_mask(flash_colreduce(q, k, "sum", True), kept)
    counts = cache_keep(cache, table, lengths, keep, pruned, pruned_table)
    out = tree_attention(query, pruned, pruned_table, counts)        # after cache_write of the drafted tokens at `counts`

The reference has none of this: its callers leave the cache to a serving program.  The kernels are csrc/cache.hip and
csrc/tree_attention.hip behind the C ABI (include/fcr.h); nothing here has a gradient.  Every call is asynchronous on the current stream of
the cache's device and allocates with torch only.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import torch

from . import _lib, flash
from .flash import _DTYPES, _raw_stream

__all__ = ["KVCache", "cache_write", "cache_read", "cache_keep", "tree_attention"]

_CODES = {torch.int8: _lib.DTYPE_INT8, torch.float8_e4m3fn: _lib.DTYPE_E4M3}
_CACHED = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, **_CODES}


class KVCache(NamedTuple):
    """Pages of keys and values: k and v are (pages, heads, page_size, D), of fp16 or bf16, or of int8 or float8_e4m3fn codes,
    which need k_scale and v_scale, fp32 (pages, heads, page_size): a row stands for its codes times its scale.

    D is a multiple of 16 up to 256, page_size a multiple of 16 (one page per sequence is a cache that is not paged).  The tensors may
    be views (keys and values in one allocation, pages of token-major rows) as far as include/fcr.h describes; a cache that is written may not be an
    expanded one, nor one whose keys and values share memory.  A page number of a table
    that is negative or not below `pages` is not there: nothing is written to it, its rows read as zeros, nothing attends to its keys."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def zeros(cls, pages: int, heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "KVCache":
        if dtype not in _CACHED:
            raise ValueError(f"A cache holds float16, bfloat16, int8 or float8_e4m3fn. Got {dtype}.")
        shape = (pages, heads, page_size, head_dim)
        k, v = (torch.zeros(shape, device=device, dtype=dtype) for _ in range(2))
        if dtype not in _CODES:
            return cls(k, v)
        return cls(k, v, *(torch.zeros(shape[:3], device=device, dtype=torch.float32) for _ in range(2)))


class _Cache(ctypes.Structure):   # fcr_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("k_strides", ctypes.c_int64 * 3), ("v_strides", ctypes.c_int64 * 3),
                ("k_scale_strides", ctypes.c_int64 * 3), ("v_scale_strides", ctypes.c_int64 * 3),
                ("dtype", ctypes.c_int), ("pages", ctypes.c_int), ("H", ctypes.c_int), ("page_size", ctypes.c_int),
                ("D", ctypes.c_int)]


def _host():
    """csrc/host.cpp: answers the calls that need neither a copy nor a message, and None to all others."""
    return flash._native or flash._host()


_I64x2 = ctypes.c_int64 * 2
_I64x3 = ctypes.c_int64 * 3


def _check_cache(cache: KVCache, name: str = "cache") -> torch.device:
    k, v = cache.k, cache.v
    if not k.is_cuda:
        raise ValueError(f"The {name} must be on CUDA device.")
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _CACHED or v.device != k.device:
        raise ValueError(f"The {name}'s keys and values must be (pages, heads, page_size, D) of one float16, bfloat16, int8 or "
                         f"float8_e4m3fn type on one device. Got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}.")
    pages, heads, page_size, d = k.shape
    if k.stride(3) != 1 or cache.v.stride(3) != 1:
        raise ValueError(f"The elements of a row of the {name} must be consecutive.")
    if max(k.shape) >= 2**31 or pages < 1 or heads < 1 or page_size < 16 or page_size % 16 or d < 16 or d > 256 or d % 16:
        raise ValueError(f"The {name} needs pages of a multiple of 16 rows, and D a multiple of 16 up to 256. Got {tuple(k.shape)}.")
    for x in (cache.k_scale, cache.v_scale):
        if k.dtype in _CODES:
            if x is None or x.shape != k.shape[:3] or x.dtype != torch.float32 or x.device != k.device:
                raise ValueError(f"The {name}'s scales must be float32 {tuple(k.shape[:3])} on its device.")
        elif x is not None:
            raise ValueError(f"The {name} holds {k.dtype}, which has no scales.")
    return k.device


def _check_table(table, device, b, name="table"):
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != b or table.device != device or \
            (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{name} must be int32 (B, pages per sequence) with B = {b} on the cache's device, unit last stride. "
                         f"Got {tuple(table.shape)} {table.dtype}.")


def _check_lengths(x, device, b, h, name):
    if x.dtype != torch.int32 or x.device != device or (x.shape != (b,) and x.shape != (b, h)):
        raise ValueError(f"{name} must be int32 ({b},) or ({b}, {h}) on the cache's device. Got {tuple(x.shape)} {x.dtype}.")


def _strides2(x):
    return _I64x2(x.stride(0), x.stride(1) if x.dim() == 2 else 0)


def _described(cache: KVCache) -> _Cache:
    k, v = cache.k, cache.v
    c = _Cache(k.data_ptr(), v.data_ptr())
    c.k_strides, c.v_strides = _I64x3(*k.stride()[:3]), _I64x3(*v.stride()[:3])
    if k.dtype in _CODES:
        c.k_scale, c.v_scale = cache.k_scale.data_ptr(), cache.v_scale.data_ptr()
        c.k_scale_strides, c.v_scale_strides = _I64x3(*cache.k_scale.stride()), _I64x3(*cache.v_scale.stride())
    c.dtype = _CACHED[k.dtype]
    c.pages, c.H, c.page_size, c.D = k.shape
    return c


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with what the C ABI asks of operands that are only read: unit d stride, 16-byte aligned rows."""
    al = 16 // x.element_size()
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0 and all(x.shape[i] == 1 or x.stride(i) % al == 0 for i in range(3)):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def cache_write(cache: KVCache, key: torch.Tensor, value: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
                counts: Optional[torch.Tensor] = None) -> None:
    """Writes key and value (B, H, T, D), fp16, bf16 or fp32, into the cache: token t of sequence b goes to position start[b] + t,
    which is row position % page_size of page table[b, position // page_size].

    int8 caches hold a row x as rint(127 x / a) with scale a / 127, float8_e4m3fn ones as the nearest such float of 448 x / a with scale a / 448,
    a = max |x_d| (ties to even); 16-bit caches hold x rounded.  A row with an infinity or a NaN reads back as NaN from a cache of
    codes.  table is int32 (B, pages per sequence); start and counts are int32 (B,), or (B, H) where the heads of a
    sequence differ in length.  With counts only the first counts[b] tokens are written.  Positions outside the table, or on a page
    that is not there, are skipped.  No row may be the place of two tokens (a page shared between sequences must not be written).
    At most 2^31 - 256 rows times D / 16 (rounded up to a power of two) in one call."""
    if _host().cache_write(cache, key, value, table, start, counts):
        return
    dev = _check_cache(cache)
    h, d = cache.k.shape[1], cache.k.shape[3]
    if key.dim() != 4 or key.shape != value.shape or key.shape[1] != h or key.shape[3] != d or key.device != dev or value.device != dev:
        raise ValueError(f"key and value must be (B, {h}, T, {d}) on the cache's device. Got {tuple(key.shape)} and {tuple(value.shape)}.")
    if key.dtype != value.dtype or key.dtype not in _DTYPES:
        raise ValueError(f"key and value must both be float16, bfloat16 or float32. Got {key.dtype} and {value.dtype}.")
    b, _, t, _ = key.shape
    _check_table(table, dev, b)
    _check_lengths(start, dev, b, h, "start")
    if counts is not None:
        _check_lengths(counts, dev, b, h, "counts")
    if b * t * table.shape[1] == 0:
        return
    key, value = _rows(key), _rows(value)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().fcr_cache_write(
            ctypes.byref(_described(cache)), table.data_ptr(), table.stride(0), table.shape[1], start.data_ptr(), _strides2(start),
            None if counts is None else counts.data_ptr(), None if counts is None else _strides2(counts), key.data_ptr(),
            value.data_ptr(), _DTYPES[key.dtype], b, t, _lib.strides4(key.stride()), _lib.strides4(value.stride()), _raw_stream(dev)))


def cache_read(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, n: int, *, out_dtype: Optional[torch.dtype] = None):
    """Positions 0 .. n-1 of every sequence and head as (key, value), each a contiguous (B, H, n, D) of out_dtype (fp16, bf16 or fp32; by
    default the cache's type, bf16 for codes), the form that flash_colreduce takes.  A code times its scale is formed in fp32 and rounded
    once.  Rows from lengths[b] (or lengths[b, h]) on are zeros.  At most 2^31 - 256 rows times D / 16 (rounded up to a power of two) in one call."""
    kv = _host().cache_read(cache, table, lengths, n, out_dtype)
    if kv is not None:
        return kv
    dev = _check_cache(cache)
    _, h, _, d = cache.k.shape
    b = table.shape[0] if table.dim() == 2 else -1
    _check_table(table, dev, b)
    _check_lengths(lengths, dev, b, h, "lengths")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if cache.k.dtype in _CODES else cache.k.dtype
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be float16, bfloat16 or float32. Got {out_dtype}.")
    if n < 0:
        raise ValueError(f"n must be >= 0. Got {n}.")
    k, v = (torch.empty((b, h, n, d), device=dev, dtype=out_dtype) for _ in range(2))
    if b * n == 0:
        return k, v
    if table.shape[1] == 0:
        return k.zero_(), v.zero_()
    with torch.cuda.device(dev):
        _lib.check(_lib.load().fcr_cache_read(
            ctypes.byref(_described(cache)), table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(), _strides2(lengths),
            k.data_ptr(), v.data_ptr(), _DTYPES[out_dtype], b, n, _raw_stream(dev)))
    return k, v


def cache_keep(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, keep: torch.Tensor, into: KVCache,
               into_table: torch.Tensor) -> torch.Tensor:
    """Keeps the rows that a mask names, each head its own: the r-th kept position of (b, h) goes, codes and scales as they are, to
    position r of into_table in `into`.  Returns how many were kept, int32 (B, H).

    keep is bool (B, H, N), as topk_keep_mask gives it for the scores of flash_colreduce; positions from lengths on, and those on a page
    that is not there, are not kept.  `into` has the cache's type, heads and D, and may be the same cache; into_table must name no page
    that `table` names.  What does not fit into_table is dropped; rows behind the kept ones are left as they were."""
    counts = _host().cache_keep(cache, table, lengths, keep, into, into_table)
    if counts is not None:
        return counts
    dev = _check_cache(cache)
    if _check_cache(into, "cache to keep rows in") != dev:
        raise ValueError("Both caches must be on the same device.")
    _, h, _, d = cache.k.shape
    if into.k.dtype != cache.k.dtype or into.k.shape[1] != h or into.k.shape[3] != d:
        raise ValueError(f"Both caches must have the same type, heads and D. Got {tuple(cache.k.shape)} {cache.k.dtype} and "
                         f"{tuple(into.k.shape)} {into.k.dtype}.")
    b = table.shape[0] if table.dim() == 2 else -1
    _check_table(table, dev, b)
    _check_table(into_table, dev, b, "into_table")
    _check_lengths(lengths, dev, b, h, "lengths")
    if keep.dtype != torch.bool or keep.dim() != 3 or keep.shape[:2] != (b, h) or keep.device != dev:
        raise ValueError(f"keep must be bool ({b}, {h}, N) on the cache's device. Got {tuple(keep.shape)} {keep.dtype}.")
    n = keep.shape[2]
    if into.k.data_ptr() == cache.k.data_ptr() and into_table.data_ptr() == table.data_ptr() and b > 0 and table.shape[1] > 0:
        raise ValueError("Rows cannot be kept in place: into_table must name other pages than table.")
    if b * n * table.shape[1] * into_table.shape[1] == 0:
        return torch.zeros((b, h), device=dev, dtype=torch.int32)
    counts = torch.empty((b, h), device=dev, dtype=torch.int32)
    keep = keep.contiguous()
    with torch.cuda.device(dev):
        _lib.check(_lib.load().fcr_cache_keep(
            ctypes.byref(_described(cache)), table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(), _strides2(lengths),
            keep.data_ptr(), n, ctypes.byref(_described(into)), into_table.data_ptr(), into_table.stride(0), into_table.shape[1],
            counts.data_ptr(), b, _raw_stream(dev)))
    return counts


@functools.lru_cache(maxsize=4096)
def _tree_bytes(dev_index: int, b: int, h: int, g: int, t: int, d: int, positions: int) -> int:
    with torch.cuda.device(dev_index):
        return _lib.load().fcr_tree_attention_bytes(b, h, g, t, d, positions)


def tree_attention(query: torch.Tensor, cache: KVCache, table: torch.Tensor, context: torch.Tensor,
                   tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, *,
                   tree_lengths: Optional[torch.Tensor] = None, return_lse2: bool = False):
    """Attention of T drafted tokens per sequence over a cache that holds their keys and values at positions context .. context+T-1.

    query is (B, Hq, T, D), fp16 or bf16 (the cache's type if that is one of them), Hq a multiple of the cache's heads: heads h*G .. h*G+G-1 attend to
    head h.  Token t sees the first context[b] (or context[b, h]) positions, and of the drafted tokens those u with tree_mask[t, u] (bool
    (T, T), or (B, T, T)): itself and its ancestors in the tree, as a rule; without a mask u <= t.  A single token is T = 1.  scale defaults to
    1/sqrt(D).  tree_lengths, int32 (B,): sequences that have fewer than T drafted tokens.

    Returns (B, Hq, T, D) of query's type, and with return_lse2 the base-2 log-sum-exp of every row's scores, fp32 (B, Hq, T), as row_lse2 has it.
    A row that sees nothing (or that the sequence does not have, or whose every score is -inf) is zeros, its log-sum-exp -inf.  What hidden rows of the
    cache hold, NaNs included, has no influence.  Probabilities are rounded to fp16 (bf16 against a bf16 cache) as they multiply the values, sums are fp32.
    The last bits of a sequence's result depend on how the work was cut, and so on the lengths of the others in the batch."""
    out = _host().tree_attention(query, cache, table, context, tree_mask, scale, tree_lengths, return_lse2)
    if out is not None:
        return out
    dev = _check_cache(cache)
    _, h, page_size, d = cache.k.shape
    if query.dim() != 4 or query.shape[3] != d or query.shape[1] % h or query.shape[1] == 0 or query.device != dev:
        raise ValueError(f"query must be (B, a multiple of {h}, T, {d}) on the cache's device. Got {tuple(query.shape)}.")
    if query.dtype not in (torch.float16, torch.bfloat16) or (cache.k.dtype not in _CODES and cache.k.dtype != query.dtype):
        raise ValueError(f"query must be float16 or bfloat16, and of the type of a cache of either. Got {query.dtype} and {cache.k.dtype}.")
    b, hq, t, _ = query.shape
    _check_table(table, dev, b)
    _check_lengths(context, dev, b, h, "context")
    if tree_mask is not None and (tree_mask.dtype != torch.bool or tree_mask.device != dev or
                                  (tree_mask.shape != (t, t) and tree_mask.shape != (b, t, t))):
        raise ValueError(f"tree_mask must be bool ({t}, {t}) or ({b}, {t}, {t}) on the cache's device. "
                         f"Got {tuple(tree_mask.shape)} {tree_mask.dtype}.")
    if tree_lengths is not None and (tree_lengths.dtype != torch.int32 or tree_lengths.shape != (b,) or tree_lengths.device != dev):
        raise ValueError(f"tree_lengths must be int32 ({b},) on the cache's device. Got {tuple(tree_lengths.shape)} {tree_lengths.dtype}.")
    if scale is None:
        scale = 1 / math.sqrt(d)
    out = torch.empty((b, hq, t, d), device=dev, dtype=query.dtype)
    lse = torch.empty((b, hq, t), device=dev, dtype=torch.float32) if return_lse2 else None
    if b * t * table.shape[1] == 0:
        out.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
        return (out, lse) if return_lse2 else out
    query = _rows(query)
    mask = None if tree_mask is None else tree_mask.contiguous()
    tree_lengths = None if tree_lengths is None else tree_lengths.contiguous()
    nbytes = _tree_bytes(dev.index if dev.index is not None else torch.cuda.current_device(), b, h, hq // h, t, d,
                         table.shape[1] * page_size)
    ws = torch.empty(max(nbytes, 16), device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().fcr_tree_attention(
            query.data_ptr(), ctypes.byref(_described(cache)), table.data_ptr(), table.stride(0), table.shape[1], context.data_ptr(),
            _strides2(context), None if mask is None else mask.data_ptr(), t * t if mask is not None and mask.dim() == 3 else 0,
            None if tree_lengths is None else tree_lengths.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(),
            ws.data_ptr(), nbytes, _DTYPES[query.dtype], b, hq // h, t, _lib.strides4(query.stride()), float(scale), _raw_stream(dev)))
    return (out, lse) if return_lse2 else out
