"""Attention over the pages of a long cache (kvcache.py) that matter to a token, chosen by a cheap score: what a step reads
of the cache no longer grows with the context.

  bounds = PageBounds(cache)
  bounds.update(table, start, count)     after tokens were written: the bounds of the pages they complete
  sparse_attention(q, cache, bounds, table, lengths, keep, ...)

A page's bounds are the smallest and largest of each element of its keys, per head. Its score for a token is the sum over
the query heads that share a cached head of sum_d max(q_d smallest_d, q_d largest_d), where a q_d of 0 counts nothing but
beside a NaN: no key of the page has a larger sum of products with them. Of the pages that hold positions up to its own, a
token keeps the `first` and the `last` ones (the last is its own page, which may be incomplete) and the best-scoring others,
`keep` in all, for each cached head; equal scores go to the lower page. A page whose score is NaN is kept first, one that is no page of the cache last (its keys are masked).

Scores are computed in 64 bits, so the choice does not depend on the order of sums. The attention over the kept pages is tree
attention's (tree.py), with the same rounding. There is no backward pass; everything runs on the current stream, lengths
and widths are read on the device only. csrc/sparse.hip has the kernels."""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from .kvcache import KVCache, check_table, padded, refuse_gradients
from .lib import Entry, Lib, float32
from .tree import DTYPES, _check

MOST_PAGES = 32768  # of a sequence
MOST_KEPT = 1024


@functools.lru_cache(maxsize=None)
def _entries() -> tuple[Entry, Entry]:
    return (Entry(name="ng_page_bounds", types="ppqiiiipqipiip"),
            Entry(name="ng_sparse_attention", types="pqqqipppppqiipqippiiiiiiiifpppp"))


@functools.lru_cache(maxsize=1024)
def _work(*shape: int) -> int:
    n = Lib().size("ng_sparse_work", *shape)
    if n < 0:
        B, T, H, G, dim, width, page, keep = shape
        raise ValueError(f"{B} sequences of {T} tokens, {H} heads x {G}, tables of {width} pages of {page}, {keep} kept: out of "
                         f"range (at most {MOST_PAGES} pages and 2^30 tokens a table, {MOST_KEPT} kept)")
    return n


class PageBounds:
    """The bounds of a cache's pages: bfloat16 [pages, heads, 2, row] (smallest, largest; rounded away from each other, zeros
    behind dim), in a tensor of its own or the given one. Only pages that update has completed hold any."""

    def __init__(self, cache: KVCache, bounds: torch.Tensor | None = None):
        shape = (cache.pages, cache.heads, 2, padded(cache.dim))
        if bounds is None:
            bounds = torch.zeros(shape, dtype=torch.bfloat16, device=cache.k.device)
        elif (bounds.shape != shape or bounds.dtype != torch.bfloat16 or bounds.get_device() != cache.device
              or not bounds.is_contiguous() or bounds.data_ptr() % 16 or bounds.requires_grad):
            raise ValueError(f"bounds must be contiguous bfloat16 {shape} on {cache.k.device}, without gradients")
        self.cache, self._bounds = cache, bounds

    bounds = property(lambda self: self._bounds, doc="bfloat16 [pages, heads, 2, row]: smallest and largest")

    def update(self, table: torch.Tensor, start: torch.Tensor, count: int) -> None:
        """The bounds of the pages that positions start[b] .. start[b] + count - 1 (start int32 [B]) lie in and that end with
        the last of them or before, from the keys the cache holds: called after a write of those positions. A page that is
        not full needs none: it is its sequence's last, which is always kept."""
        c = self.cache
        check_table(c, table)
        B, width = table.shape
        start = _check("start", start, (B,), torch.int32, c)
        if not 0 <= count < 1 << 30:
            raise ValueError(f"count must be 0 to 2^30 - 1: {count}")
        k, _, ks, _ = c.addresses()
        _entries()[0](c.device, k, ks, c.pages, c.page, c.heads, c.dim, c.code, table.data_ptr(), table.stride(0), width,
                      start.data_ptr(), B, count, self._bounds.data_ptr())


def sparse_attention(q: torch.Tensor, cache: KVCache, bounds: PageBounds, table: torch.Tensor, lengths: torch.Tensor, keep: int,
                     widths: torch.Tensor | None = None, first: int = 1, last: int = 1, scale: float | None = None,
                     return_lse: bool = False, return_pages: bool = False):
    """Attention of q [B, T, heads * group, dim] (bfloat16 or float16, a 16-bit cache's own type; any strides over the first
    three) over each token's kept pages; token t of sequence b stands at position lengths[b] + t and sees the positions up to
    its own, whose keys and values are written already. Query head h reads the cache's head h // group.

    table    int32 [B, width]: the sequences' pages in order (at most 32768); keys whose entry is no page of the cache are masked
    lengths  int32 [B]: the tokens before q's (held to 0 .. what the table covers)
    keep     pages kept of those a token sees, first + last of them at least (1 to 1024)
    widths   int32 [B]: the tokens in use (None: all T); the rows past them are zeros, whatever q holds there
    first    the sequence's first pages, always kept; last: its last ones up to the token's own, 1 at least
    scale    the scores' factor, 1 / sqrt(dim) by default

    Returns the output in q's shape and type; with return_lse also the float32 [B, T, heads * group] logarithms of the softmax
    sums (-inf where a row sees nothing, whose output is zeros), with return_pages also int32 [B, T, cache heads, keep], the
    kept pages' places in the sequence in order, -1 behind them."""
    size, dtype = q.shape, q.dtype
    if len(size) != 4 or dtype not in DTYPES:
        raise ValueError(f"q must be [B, T, heads, dim] in bfloat16 or float16: got {tuple(size)} {dtype}")
    B, T, heads, dim = size
    if dim != cache.dim or heads < 1 or heads % cache.heads or T < 1:
        raise ValueError(f"q {tuple(size)} does not go with {cache.heads} cached heads of {cache.dim}: a multiple of the "
                         "heads, at least one token")
    if cache.code >= 2 and dtype != cache.k.dtype:
        raise ValueError(f"a {cache.k.dtype} cache takes queries of its own type: got {dtype}")
    if q.get_device() != cache.device:
        raise ValueError(f"q is on {q.device}, the cache on {cache.k.device}")
    if bounds.cache is not cache:
        raise ValueError("the bounds are another cache's")
    if q.requires_grad or forward_ad._current_level >= 0:
        refuse_gradients("sparse_attention", q)
    check_table(cache, table)
    tables, width = table.shape
    if tables != B:
        raise ValueError(f"{tables} page tables for {B} sequences")
    if not 1 <= keep <= MOST_KEPT or first < 0 or last < 1 or first + last > keep:
        raise ValueError(f"keep must be 1 to {MOST_KEPT} pages, the first and at least one last of them among these: "
                         f"{keep}, {first}, {last}")
    lengths = _check("lengths", lengths, (B,), torch.int32, cache)
    if widths is not None:
        widths = _check("widths", widths, (B,), torch.int32, cache)
    scale = 1 / math.sqrt(dim) if scale is None else float32("scale", scale)
    qb, qt, qh, qd = q.stride()
    if qd != 1:  # (of one element a row, too, which torch calls contiguous and may have negated by a bit alone)
        q = q.resolve_neg().contiguous()
        qb, qt, qh, _ = q.stride()
    device, group = cache.k.device, heads // cache.heads
    work = torch.empty(_work(B, T, cache.heads, group, dim, width, cache.page, keep), dtype=torch.uint8, device=device)
    out = torch.empty(size, dtype=dtype, device=device)
    lse = torch.empty(size[:3], dtype=torch.float32, device=device) if return_lse else None
    pages = torch.empty((B, T, cache.heads, keep), dtype=torch.int32, device=device) if return_pages else None
    k, v, ks, vs = cache.addresses()
    _entries()[1](cache.device, q.data_ptr(), qb, qt, qh, DTYPES[dtype], k, v, ks, vs, bounds.bounds.data_ptr(), cache.pages,
                  cache.page, cache.code, table.data_ptr(), table.stride(0), width, lengths.data_ptr(),
                  None if widths is None else widths.data_ptr(), B, T, cache.heads, group, dim, keep, first, last, scale,
                  out.data_ptr(), None if lse is None else lse.data_ptr(), None if pages is None else pages.data_ptr(),
                  work.data_ptr())
    more = [x for x in (lse, pages) if x is not None]
    return (out, *more) if more else out
