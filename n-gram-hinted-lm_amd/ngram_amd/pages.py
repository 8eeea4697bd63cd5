"""Who holds the pages of a paged cache (kvcache.py): sequences that fork share the pages of what they have in common, a page
is copied only where one of them goes on writing it, and what nobody holds is free again.

  pool = PagePool(cache)                        every page free
  pool.hold(table)                              a table made elsewhere: its entries counted
  pool.fork(table, lengths, parents)            row s becomes what row parents[s] was; below 0: empty, its pages let go
  slots = pool.reserve(table, lengths, count)   room for count more tokens a row, as the slots that KVCache.write takes
  table = pool.move(table, into)                the pages in use, packed into another pool's cache
  copy_pages(cache, other, pages, others)       pages of one cache to another

Tables are int32 [rows, width], a row's pages in order and -1 behind them; lengths int32 [rows], the tokens that each row
holds. Both are changed in place, so that captured graphs find them where they were; lengths only by a fork (the caller adds
what it has written). Every table's entries must be counted: by hold, by a fork or by a reservation.

Pages and counts are whole numbers and choices go by order (the lowest free pages, in the order of rows), so the same calls
give the same pages on every run. Everything runs on the current stream and nothing synchronizes: where the pages do not
suffice, `missing` on the device counts the ones that were not to be had, and their positions' slots are -1. A pool is one
state: calls on it from several streams must be ordered by the caller. csrc/pages.hip has the kernels."""

from __future__ import annotations

import functools

import torch

from .kvcache import KVCache, check_table
from .lib import Entry, Lib


@functools.lru_cache(maxsize=None)
def _entries() -> tuple[Entry, ...]:
    return (Entry(name="ng_pool_clear", types="pq"), Entry(name="ng_pool_hold", types="pqpqii"),
            Entry(name="ng_pool_fork", types="pqpqiippp"), Entry(name="ng_pool_room", types="pqpqiippippppiiiipp"),
            Entry(name="ng_pool_move", types="pqppppppqpppppiiiipqiipp"),
            Entry(name="ng_copy_pages", types="pppppqpppppqiiiippq"))


@functools.lru_cache(maxsize=1024)
def _size(name: str, *args: int) -> int:
    n = Lib().size("ng_" + name, *args)
    if n < 0:
        raise ValueError(f"{name} of {args}: out of range")
    return n


class PagePool:
    """The pages of a KVCache; with bounds (sparse.PageBounds over the same cache) a move takes those along."""

    def __init__(self, cache: KVCache, bounds=None):
        if bounds is not None and bounds.cache is not cache:
            raise ValueError("the bounds are another cache's")
        self.cache, self.bounds = cache, bounds
        self._state = torch.empty(_size("pool_state", cache.pages) // 4, dtype=torch.int32, device=cache.k.device)
        self.clear()

    # refs: the entries that hold each page. missing: pages that reservations and moves did not get, since the pool was cleared.
    refs = property(lambda self: self._state[:self.cache.pages], doc="int32 [pages]: the table entries that hold each page")
    missing = property(lambda self: self._state[-1:], doc="int32 [1]: the pages that were not to be had")

    def clear(self) -> None:
        """Every page free."""
        _entries()[0](self.cache.device, self._state.data_ptr(), self.cache.pages)

    def _rows(self, table: torch.Tensor, lengths: torch.Tensor | None = None) -> tuple[int, int]:
        check_table(self.cache, table)
        S, width = table.shape
        if S > 1 and table.stride(0) < width:
            raise ValueError("the page table's rows overlap")
        if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != (S,) or
                                    lengths.get_device() != self.cache.device or not lengths.is_contiguous()):
            raise ValueError(f"lengths must be contiguous int32 [{S}] on {self.cache.k.device}")
        return S, width

    def hold(self, table: torch.Tensor) -> None:
        """The entries of a table made elsewhere, counted: its pages are no longer free."""
        S, width = self._rows(table)
        _entries()[1](self.cache.device, self._state.data_ptr(), self.cache.pages, table.data_ptr(), table.stride(0), S, width)

    def fork(self, table: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor) -> None:
        """Row s of the table and the lengths becomes what row parents[s] was (int64 [rows], or any shape of as many: a
        BeamStep's); a parent that is no row leaves it empty: length 0, entries -1. Pages are shared, not copied."""
        S, width = self._rows(table, lengths)
        if parents.dtype != torch.int64 or parents.numel() != S or parents.get_device() != self.cache.device:
            raise ValueError(f"parents must be int64 of {S} rows on {self.cache.k.device}: got {tuple(parents.shape)} "
                             f"{parents.dtype} on {parents.device}")
        parents = parents.contiguous()
        size = _size("pool_fork_work", S, width)
        work = torch.empty(size, dtype=torch.uint8, device=table.device) if size else None
        _entries()[2](self.cache.device, self._state.data_ptr(), self.cache.pages, table.data_ptr(), table.stride(0), S, width,
                      lengths.data_ptr(), parents.data_ptr(), None if work is None else work.data_ptr())

    def reserve(self, table: torch.Tensor, lengths: torch.Tensor, count: int, counts: torch.Tensor | None = None) -> torch.Tensor:
        """Room behind each row's tokens for `count` more (or counts[s], int32 [rows], held to 0 .. count): int64 [rows,
        count], their slots, -1 past a row's own count, past the table and where no page was to be had (`missing`). A page
        that others hold is left to them: the row gets another, with a copy of the rows before its length; where all that
        hold it ask in this call, the longest of them keeps it, of equal ones the first, so that what it writes lies behind
        the tokens of a row that gets none and is left with the shared page."""
        S, width = self._rows(table, lengths)
        if not 0 <= count < 1 << 30:
            raise ValueError(f"count must be 0 to 2^30 - 1: {count}")
        c = self.cache
        if counts is not None:
            if counts.dtype != torch.int32 or counts.shape != (S,) or counts.get_device() != c.device:
                raise ValueError(f"counts must be int32 [{S}] on {c.k.device}")
            counts = counts.contiguous()
        slots = torch.empty((S, count), dtype=torch.int64, device=table.device)
        if S and count:
            work = torch.empty(_size("pool_room_work", S, count, c.page), dtype=torch.uint8, device=table.device)
            _entries()[3](c.device, self._state.data_ptr(), c.pages, table.data_ptr(), table.stride(0), S, width,
                          lengths.data_ptr(), None if counts is None else counts.data_ptr(), count, *c.addresses(), c.page,
                          c.heads, c.dim, c.code, slots.data_ptr(), work.data_ptr())
        return slots

    def move(self, table: torch.Tensor, into: "PagePool") -> torch.Tensor:
        """This pool's pages in use, in order, into the first pages of another pool's cache (of the same heads, dim, page size
        and codes; any number of pages), which holds nothing else afterwards: its counts are this pool's. Returns the table
        with the pages' new numbers (-1 where it had no room: into.missing); other tables over this pool are moved with
        the same call on tables joined beforehand. This pool and its tables are left as they are."""
        a, b = self.cache, into.cache
        S, width = self._rows(table)
        _check_alike(a, b)
        if into is self or b is a or a.k.data_ptr() == b.k.data_ptr():
            raise ValueError("a pool is moved into another cache's")
        if (self.bounds is None) != (into.bounds is None):
            raise ValueError("both pools need bounds, or neither")
        out = torch.empty((S, width), dtype=torch.int32, device=table.device)
        work = torch.empty(_size("pool_move_work", a.pages, b.pages), dtype=torch.uint8, device=table.device)
        _entries()[4](a.device, self._state.data_ptr(), a.pages, *a.addresses(), _bounds(self.bounds), into._state.data_ptr(),
                      b.pages, *b.addresses(), _bounds(into.bounds), a.page, a.heads, a.dim, a.code, table.data_ptr(),
                      table.stride(0), S, width, out.data_ptr(), work.data_ptr())
        return out


def _bounds(bounds) -> int | None:
    return None if bounds is None else bounds.bounds.data_ptr()


def _check_alike(a: KVCache, b: KVCache) -> None:
    if (a.page, a.heads, a.dim, a.code, a.device) != (b.page, b.heads, b.dim, b.code, b.device):
        raise ValueError(f"caches of {(a.page, a.heads, a.dim, a.k.dtype, a.k.device)} and "
                         f"{(b.page, b.heads, b.dim, b.k.dtype, b.k.device)} (page, heads, dim, codes, device) differ")


def copy_pages(cache: KVCache, other: KVCache, pages: torch.Tensor, others: torch.Tensor, bounds=None, other_bounds=None) -> None:
    """Page others[i] of the cache `other` becomes what page pages[i] of `cache` is (int64 [n] each; a pair with a number that is
    no page is passed over), with their bounds (sparse.PageBounds of each) where those are given. Within one cache no page
    may be both read and written; a page given twice in `others` is left with a mixture."""
    _check_alike(cache, other)
    for name, p in (("pages", pages), ("others", others)):
        if p.dtype != torch.int64 or p.dim() != 1 or p.shape != pages.shape or p.get_device() != cache.device:
            raise ValueError(f"{name} must be int64 [n] on {cache.k.device}: got {tuple(p.shape)} {p.dtype} on {p.device}")
    if (bounds is None) != (other_bounds is None) or (bounds is not None and (bounds.cache is not cache or
                                                                             other_bounds.cache is not other)):
        raise ValueError("bounds must be given for both caches, each its own")
    pages, others = pages.contiguous(), others.contiguous()
    _entries()[5](cache.device, *cache.addresses(), _bounds(bounds), cache.pages, *other.addresses(), _bounds(other_bounds),
                  other.pages, cache.page, cache.heads, cache.dim, cache.code, pages.data_ptr(), others.data_ptr(),
                  pages.shape[0])
