"""What a caller that drafts tokens does after the target model's step: which of them stand and what comes next (verify_drafts), their rows moved
to where they belong (cache_accept), and room for the next ones (cache_reserve).

    granted = cache_reserve(pool, table, context + T, page_size)              # pages for T drafted tokens
    cache_write(cache, key, value, table, context)
    out = tree_attention(query, cache, table, context, tree_mask)             # ... the model's probabilities behind every token
    accepted, path, token = verify_drafts(target, tokens, uniform, sample, parents=parents)
    context = cache_accept(cache, table, context, path, accepted)             # each layer's cache
    cache_reserve(pool, table, context, page_size)                            # pages of what was rejected go back

Models that cap their scores, bias them by distance or limit them to a window attend to a drafted chain by chunk_attention; tree_attention, which trees need, has plain
scores only.

The reference has none of this.  The kernels are csrc/drafts.hip behind the C ABI (include/fcr.h); nothing here has a gradient.  Every call is
asynchronous on the current stream of its operands' device and allocates with torch only; all of them can be captured into a graph.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .cache import KVCache, _check_cache, _check_lengths, _check_table, _described, _host, _I64x2, _strides2
from .flash import _DTYPES, _raw_stream

__all__ = ["Verified", "PagePool", "verify_drafts", "cache_accept", "cache_reserve"]


class Verified(NamedTuple):
    """accepted: int32 (B,), how many drafted tokens stand.  path: int32 (B, T), which ones, in their order, then -1.  token: (B,), the one behind them."""
    accepted: torch.Tensor
    path: torch.Tensor
    token: torch.Tensor


def _check_ints(x, shape, device, name):
    if x.dtype != torch.int32 or tuple(x.shape) != shape or x.device != device:
        raise ValueError(f"{name} must be int32 {shape} on the same device. Got {tuple(x.shape)} {x.dtype}.")


def _check_probabilities(x, shape, dtype, device, name):
    if x.dim() != 3 or tuple(x.shape) != shape or x.dtype != dtype or x.device != device:
        raise ValueError(f"{name} must be {dtype} {shape} on the same device. Got {tuple(x.shape)} {x.dtype}.")


def _in_rows(x: torch.Tensor) -> torch.Tensor:
    return x if (x.shape[2] == 1 or x.stride(2) == 1) and min(x.stride()) >= 0 else x.contiguous()


def verify_drafts(target: torch.Tensor, tokens: torch.Tensor, uniform: torch.Tensor, sample: torch.Tensor, *,
                  draft: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None,
                  counts: Optional[torch.Tensor] = None) -> Verified:
    """Which drafted tokens stand, so that what comes out is distributed as the target draws it, from given random numbers.

    target: (B, T+1, V) probabilities, fp32, fp16 or bf16; row 0 is the distribution behind the context, row i+1 the one behind token i.  tokens: (B, T), int32 or
    int64.  parents: int32 (T,) or (B, T), which token each one continues, an earlier one, or the context (-1); without it the tokens are a chain.  counts:
    int32 (B,), sequences that have fewer than T.  uniform: fp32 (B, T) and sample: fp32 (B,), numbers in [0, 1).  T may be 0, at most 1024.

    With draft, (B, T, V) of target's type, the probabilities that the tokens of a chain were drawn from: token i stands if those in front do and
    uniform[b, i] * draft[b, i, x] < target[b, i, x]; the next token is drawn from max(target - draft, 0) of the row where the path ends.
    Without (likely tokens, trees of them): the children of a row share [0, 1) by their probabilities, in their order, a token that an earlier one has already
    without a share; the one that uniform[b, row] falls to stands, and where it falls to none the next token is drawn from what the row has beside them.
    That is the first token at which the sum of what it is drawn from exceeds sample[b] of the whole, -1 where there is no weight at all or an infinite
    one.  A probability below 0, or a NaN, counts as 0; a row's probabilities need not add up to exactly 1.  Tokens outside the vocabulary, and those whose
    parent is neither -1 nor an earlier token, never stand."""
    out = _host().verify_drafts(target, tokens, uniform, sample, draft, parents, counts)
    if out is not None:
        return Verified(*out)
    if not target.is_cuda:
        raise ValueError("Probabilities must be on CUDA device.")
    dev = target.device
    if target.dim() != 3 or target.dtype not in _DTYPES or target.shape[1] < 1 or target.shape[2] < 1:
        raise ValueError(f"target must be float16, bfloat16 or float32 (B, T+1, V). Got {tuple(target.shape)} {target.dtype}.")
    b, t, v = target.shape[0], target.shape[1] - 1, target.shape[2]
    if tokens.dtype not in (torch.int32, torch.int64) or tuple(tokens.shape) != (b, t) or tokens.device != dev:
        raise ValueError(f"tokens must be int32 or int64 ({b}, {t}) on the same device. Got {tuple(tokens.shape)} {tokens.dtype}.")
    for x, shape, name in ((uniform, (b, t), "uniform"), (sample, (b,), "sample")):
        if x.dtype != torch.float32 or tuple(x.shape) != shape or x.device != dev:
            raise ValueError(f"{name} must be float32 {shape} on the same device. Got {tuple(x.shape)} {x.dtype}.")
    if draft is not None:
        if parents is not None:
            raise ValueError("Tokens that come with the probabilities that they were drawn from must be a chain: give draft or parents.")
        _check_probabilities(draft, (b, t, v), target.dtype, dev, "draft")
    if parents is not None:
        _check_ints(parents, (b, t) if parents.dim() == 2 else (t,), dev, "parents")
    if counts is not None:
        _check_ints(counts, (b,), dev, "counts")
    if t > 1024 or v > 2**28 or b > 2**20:
        raise ValueError(f"At most 1024 drafted tokens, 2^28 possible ones and 2^20 sequences. Got {t}, {v} and {b}.")
    accepted = torch.empty((b,), device=dev, dtype=torch.int32)
    path = torch.empty((b, t), device=dev, dtype=torch.int32)
    token = torch.empty((b,), device=dev, dtype=tokens.dtype)
    if b == 0:
        return Verified(accepted, path, token)
    target, tokens, uniform, sample = _in_rows(target), tokens.contiguous(), uniform.contiguous(), sample.contiguous()
    draft = None if draft is None or t == 0 else _in_rows(draft)
    parents = None if parents is None else parents.contiguous()
    counts = None if counts is None else counts.contiguous()
    with torch.cuda.device(dev):
        lib = _lib.load()
        nbytes = lib.fcr_verify_drafts_bytes(b, t, v)
        ws = torch.empty(max(nbytes, 16), device=dev, dtype=torch.uint8)
        _lib.check(lib.fcr_verify_drafts(
            target.data_ptr(), _I64x2(*target.stride()[:2]), None if draft is None else draft.data_ptr(),
            None if draft is None else _I64x2(*draft.stride()[:2]), tokens.data_ptr() or None, tokens.element_size(),
            None if parents is None else parents.data_ptr() or None, t if parents is not None and parents.dim() == 2 else 0,
            None if counts is None else counts.data_ptr(), uniform.data_ptr() or None, sample.data_ptr(), accepted.data_ptr(),
            path.data_ptr() or None, token.data_ptr(), ws.data_ptr(), nbytes, _DTYPES[target.dtype], b, t, v, _raw_stream(dev)))
    return Verified(accepted, path, token)


def cache_accept(cache: KVCache, table: torch.Tensor, context: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor) -> torch.Tensor:
    """Moves the rows of accepted tokens, in place: of sequence b the keys and values at position context + path[b, i] go to position context + i,
    i < accepted[b], in every head, codes and scales as they are.  Returns context + accepted, int32 of context's shape.

    context: int32 (B,), or (B, H) where the heads of a sequence differ in length; path: int32 (B, T) and accepted: int32 (B,), as verify_drafts gives them (a path
    rises).  Rows that would come from or go to a page that is not there, or behind the table, are left alone; so is every row behind the accepted ones.
    The cache must be one that may be written (see KVCache)."""
    moved = _host().cache_accept(cache, table, context, path, accepted)
    if moved is not None:
        return moved
    dev = _check_cache(cache)
    h = cache.k.shape[1]
    b = table.shape[0] if table.dim() == 2 else -1
    _check_table(table, dev, b)
    _check_lengths(context, dev, b, h, "context")
    if path.dim() != 2:
        raise ValueError(f"path must be int32 ({b}, T). Got {tuple(path.shape)} {path.dtype}.")
    _check_ints(path, (b, path.shape[1]), dev, "path")
    _check_ints(accepted, (b,), dev, "accepted")
    t = path.shape[1]
    if b * t * table.shape[1] == 0:
        n = accepted.clamp(0, t)
        return context.clamp_min(0) + (n if context.dim() == 1 else n[:, None])
    # (a stride of 0 in the second dimension says that heads have one length: a view of (B, H) with such a one is copied)
    out = torch.empty(context.shape, device=dev, dtype=torch.int32)
    if context.dim() == 2 and context.stride(1) == 0:
        context = context.contiguous()
    path, accepted = path.contiguous(), accepted.contiguous()
    with torch.cuda.device(dev):
        _lib.check(_lib.load().fcr_cache_accept(
            ctypes.byref(_described(cache)), table.data_ptr(), table.stride(0), table.shape[1], context.data_ptr(), _strides2(context),
            path.data_ptr(), accepted.data_ptr(), out.data_ptr(), b, t, _raw_stream(dev)))
    return out


class PagePool(NamedTuple):
    """Pages that no sequence holds, a stack: free, int32 (pages,), of which the first available, int32 (1,), lie on it; and held, int32 (B,), how
    many entries of each sequence's row of a table are its own.  One page number stands for a page of every layer's cache."""
    free: torch.Tensor
    available: torch.Tensor
    held: torch.Tensor

    @classmethod
    def full(cls, pages: int, sequences: int, device="cuda") -> "PagePool":
        """All pages free, the lowest on top; a table to go with it is torch.full((sequences, n), -1, dtype=torch.int32)."""
        return cls(torch.arange(pages - 1, -1, -1, device=device, dtype=torch.int32), torch.full((1,), pages, device=device, dtype=torch.int32),
                   torch.zeros((sequences,), device=device, dtype=torch.int32))


def cache_reserve(pool: PagePool, table: torch.Tensor, lengths: torch.Tensor, page_size: int) -> torch.Tensor:
    """Gives every sequence the pages for lengths[b] positions and takes back those that it no longer needs; table and pool are changed in place.
    Returns bool (B,): whether a sequence now holds what it needs.

    lengths: int32 (B,), or (B, H), of which the longest head counts; 0 gives all pages back.  Pages go back first, in the order of
    sequences and entries, their entries become -1; then those that need more take pages from the top of the stack, in the order of sequences, up to
    the first for which too few are left: it and all behind it that need more stay as they are, as does one that needs more than the table's
    row names.  table: int32 (B, pages per sequence), the first held[b] entries of a row its pages, rows that do not overlap.  Page numbers must be on the stack
    or in one row, and there once (pages that several rows share are not for this)."""
    granted = _host().cache_reserve(pool, table, lengths, page_size)
    if granted is not None:
        return granted
    free, available, held = pool
    if not table.is_cuda:
        raise ValueError("The table must be on CUDA device.")
    dev = table.device
    b = table.shape[0] if table.dim() == 2 else -1
    _check_table(table, dev, b)
    if b > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("The rows of a table that is written must not overlap.")
    if lengths.dtype != torch.int32 or lengths.device != dev or lengths.dim() not in (1, 2) or lengths.shape[0] != b or lengths.shape[-1] == 0 < b:
        raise ValueError(f"lengths must be int32 ({b},) or ({b}, heads) on the table's device. Got {tuple(lengths.shape)} {lengths.dtype}.")
    _check_ints(available, (1,), dev, "available")
    _check_ints(held, (b,), dev, "held")
    if free.dim() != 1 or free.dtype != torch.int32 or free.device != dev or free.shape[0] < 1:
        raise ValueError(f"free must be int32 (pages,) on the table's device. Got {tuple(free.shape)} {free.dtype}.")
    if not (free.is_contiguous() and held.is_contiguous()):
        raise ValueError("The pool's tensors must be contiguous.")
    if not 1 <= page_size or page_size * table.shape[1] > 2**30:
        raise ValueError(f"page_size must be >= 1, and a table's row name at most 2^30 positions. Got {page_size}.")
    granted = torch.empty((b,), device=dev, dtype=torch.bool)
    if b == 0:
        return granted
    if table.shape[1] == 0:
        return torch.le(lengths if lengths.dim() == 1 else lengths.amax(1), 0, out=granted)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().fcr_cache_reserve(
            table.data_ptr(), table.stride(0), table.shape[1], held.data_ptr(), free.data_ptr(), free.shape[0], available.data_ptr(),
            lengths.data_ptr(), _strides2(lengths), lengths.shape[-1] if lengths.dim() == 2 else 1, page_size, granted.data_ptr(), b,
            _raw_stream(dev)))
    return granted
