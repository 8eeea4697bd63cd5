"""A paged key/value cache that is quantised as it is written: the cache that tree attention (tree.py) reads.

Codes lie in pages, [pages, heads, page size, dim padded with zeros to a multiple of 64], in one of
  int8   code = x * (127 / a) rounded half to even, a = max |x| over a token's row of one head
  fp8    e4m3, code = x * (448 / a) rounded half to even
  bf16, fp16   x itself
and the 8-bit ones have a float32 scale a / 127 or a / 448 per token and head, [pages, heads, page size]. A row that is
zero (or too small for its inverse) has scale 0; one that holds a NaN or an infinity has codes 0 and scale NaN, so that it
reads back as NaN and nothing of it enters where it is masked. A scale of 0 stands for zeros whatever the codes are.

A token's slot is page * page size + its row there; a sequence's page table lists its pages in order, and -1 stands for no
slot. Which page belongs to whom is the caller's, or a pool's (pages.py). Quantising has no backward pass: keys and values
that require gradients (with gradients on) or carry tangents raise. Everything runs on the current stream, and nothing here
synchronizes. csrc/kvcache.hip has the kernels."""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from .lib import Entry

CODES = {torch.int8: 0, torch.float8_e4m3fn: 1, torch.bfloat16: 2, torch.float16: 3}
NAMES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16, "fp16": torch.float16}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@functools.lru_cache(maxsize=None)
def _entries() -> tuple[Entry, Entry, Entry]:
    return (Entry(name="ng_kv_write", types="ppqqqqipqppppqiiii"), Entry(name="ng_kv_read", types="ppppqiiiipqppi"),
            Entry(name="ng_kv_slots", types="pqipiiqip"))


def padded(dim: int) -> int:
    """The length of a cached row of `dim` elements."""
    return (dim + 63) // 64 * 64


def refuse_gradients(what: str, *tensors: torch.Tensor) -> None:
    """Raises where gradients would be lost: a tensor that requires one while they are on, or has a forward-mode tangent."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors) or (
            forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)):
        raise RuntimeError(f"{what} has no backward pass and its input requires a gradient: call it under torch.no_grad() or "
                           "on detached tensors")


class KVCache:
    """KVCache(k, v, k_scale, v_scale, dim) over tensors in hand, or KVCache.empty(...) with its own."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, dim: int | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in CODES:
            raise ValueError(f"k and v must both be [pages, heads, page size, row] in int8, float8_e4m3fn, bfloat16 or "
                             f"float16: got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        pages, heads, page, row = k.shape
        self.dim = row if dim is None else int(dim)
        if not 1 <= self.dim <= 256 or row != padded(self.dim):
            raise ValueError(f"rows of {row} do not hold heads of {self.dim}: 1 to 256, padded to a multiple of 64")
        if pages < 1 or heads < 1 or not 16 <= page <= 4096 or page & (page - 1):
            raise ValueError(f"{pages} pages of {page} tokens and {heads} heads: at least one, pages a power of two from "
                             "16 to 4096")
        if not (k.is_cuda and k.device == v.device and k.is_contiguous() and v.is_contiguous()):
            raise ValueError("k and v must be contiguous and on one GPU")
        if k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("k and v must start at a multiple of 16 bytes")
        if k.element_size() == 1:
            for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
                if (s is None or s.shape != (pages, heads, page) or s.dtype != torch.float32 or s.device != k.device
                        or not s.is_contiguous() or s.data_ptr() % 16):
                    raise ValueError(f"{name} must be contiguous float32 {(pages, heads, page)} beside 8-bit codes")
        elif k_scale is not None or v_scale is not None:
            raise ValueError("a 16-bit cache has no scales")
        if any(t is not None and t.requires_grad for t in (k, v, k_scale, v_scale)):
            raise ValueError("a cache's tensors take no gradients")
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page = pages, heads, page
        self.code, self.device = CODES[k.dtype], k.get_device()
        self._ptr = tuple(None if t is None else t.data_ptr for t in (k, v, k_scale, v_scale))

    # The tensors are the cache's for good (its shape is theirs): a larger or moved cache is another KVCache.
    k = property(lambda self: self._k, doc="the keys' codes [pages, heads, page size, row]")
    v = property(lambda self: self._v, doc="the values' codes [pages, heads, page size, row]")
    k_scale = property(lambda self: self._k_scale, doc="the keys' scales [pages, heads, page size], None in 16 bits")
    v_scale = property(lambda self: self._v_scale, doc="the values' scales [pages, heads, page size], None in 16 bits")

    def addresses(self) -> tuple:
        """k, v, k_scale, v_scale as the kernels take them: where they lie now."""
        k, v, ks, vs = self._ptr
        return k(), v(), ks and ks(), vs and vs()

    @classmethod
    def empty(cls, pages: int, page: int, heads: int, dim: int, codes: str = "int8",
              device: torch.device | str = "cuda") -> "KVCache":
        """A cache of zeros in its own memory."""
        if codes not in NAMES:
            raise ValueError(f"codes must be one of {sorted(NAMES)}: {codes!r}")
        dt = NAMES[codes]
        k, v = (torch.zeros((pages, heads, page, padded(dim)), dtype=torch.uint8 if dt.itemsize == 1 else dt,
                            device=device) for _ in range(2))
        scales = [torch.zeros((pages, heads, page), device=device) for _ in range(2)] if dt.itemsize == 1 else [None] * 2
        return cls(k.view(dt), v.view(dt), *scales, dim=dim)

    def _slots(self, slots: torch.Tensor, n: int) -> torch.Tensor:
        if slots.dtype != torch.int64 or slots.shape != (n,) or slots.get_device() != self.device:
            raise ValueError(f"slots must be int64 [{n}] on {self.k.device}: got {tuple(slots.shape)} {slots.dtype} on "
                             f"{slots.device}")
        return slots.contiguous()

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """The tokens' keys and values [n, heads, dim] (any strides over tokens and heads; float32, bfloat16 or float16,
        a 16-bit cache's own type) into their slots (int64 [n]); a token whose slot is negative or past the cache is not
        written. Slots given twice in one call leave either token."""
        size, dtype = k.shape, k.dtype
        if (len(size) != 3 or size[1] != self.heads or size[2] != self.dim or v.shape != size or v.dtype != dtype
                or dtype not in DTYPES):
            raise ValueError(f"k and v must both be [n, {self.heads}, {self.dim}] in float32, bfloat16 or float16: got "
                             f"{tuple(size)} {dtype} and {tuple(v.shape)} {v.dtype}")
        if self.code >= 2 and dtype != self.k.dtype:
            raise ValueError(f"a {self.k.dtype} cache takes its own type: got {dtype}")
        if k.get_device() != self.device or v.get_device() != self.device:
            raise ValueError(f"k and v must be on {self.k.device}")
        (kt, kh, kd), (vt, vh, vd) = k.stride(), v.stride()
        if kd != 1 or vd != 1:
            k, v = k.resolve_neg().contiguous(), v.resolve_neg().contiguous()
            (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
        if k.requires_grad or v.requires_grad or forward_ad._current_level >= 0:
            refuse_gradients("KVCache.write", k, v)
        slots = self._slots(slots, size[0])
        _entries()[0](self.device, k.data_ptr(), v.data_ptr(), kt, kh, vt, vh, DTYPES[dtype], slots.data_ptr(), size[0],
                      *self.addresses(), self.pages, self.page, self.heads, self.dim, self.code)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values held in slots (int64 [n]) as [n, heads, dim] of `dtype`: code * scale in 32 bits, rounded
        once; zeros where a slot is negative or past the cache."""
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be float32, bfloat16 or float16: {dtype}")
        n = slots.shape[0] if slots.dim() else 0
        slots = self._slots(slots, n)
        k = torch.empty((n, self.heads, self.dim), dtype=dtype, device=self.k.device)
        v = torch.empty_like(k)
        _entries()[1](self.device, *self.addresses(), self.pages, self.page, self.heads, self.dim, self.code,
                      slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), DTYPES[dtype])
        return k, v

    def slots(self, table: torch.Tensor, start: torch.Tensor, count: int) -> torch.Tensor:
        """int64 [B, count]: the slots of positions start[b], start[b] + 1, ... of sequences with page tables table
        (int32 [B, width]); -1 past a table or where its entry is no page of the cache. start int32 [B]."""
        check_table(self, table)
        B, width = table.shape
        if start.dtype != torch.int32 or start.shape != (B,) or start.get_device() != self.device:
            raise ValueError(f"start must be int32 [{B}] on {self.k.device}")
        if not 0 <= count < 1 << 31:
            raise ValueError(f"count must be 0 to 2^31 - 1: {count}")
        start = start.contiguous()
        out = torch.empty((B, count), dtype=torch.int64, device=self.k.device)
        _entries()[2](self.device, table.data_ptr(), table.stride(0), width, start.data_ptr(), B, count, self.pages,
                      self.page, out.data_ptr())
        return out


def check_table(cache: KVCache, table: torch.Tensor) -> None:
    if table.dtype != torch.int32 or table.dim() != 2 or table.get_device() != cache.device:
        raise ValueError(f"the page table must be int32 [sequences, width] on {cache.k.device}: got "
                         f"{tuple(table.shape)} {table.dtype} on {table.device}")
    width = table.shape[1]
    if width < 1 or (width > 1 and table.stride(1) != 1):
        raise ValueError("the page table's rows must be non-empty and contiguous")
