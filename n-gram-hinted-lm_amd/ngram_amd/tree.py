"""Attention for a tree of drafted tokens over a paged cache (kvcache.py): how a model verifies the continuations that this
package's counts and matches draft. A sequence of lengths[b] cached tokens gets up to 64 drafted ones in a step, their keys
and values written behind the cached ones (the token i of the tree at position lengths[b] + i); each sees the cached tokens
and its own ancestors, so every path of the tree is scored as if it were the sequence's continuation. One token without a
mask is ordinary decoding. There is no backward pass: queries that require gradients (with gradients on) raise.

  tree_attention(q, cache, table, lengths, mask=None, widths=None, scale=None, return_lse=False)
  tree_mask(parents)    the ancestors' bits of trees given by their parents

Scores, the softmax's sums and the outputs' are held in 32 bits; a weight is rounded to 16 bits for its product with the
values (float16, bfloat16 over a bfloat16 cache), as an output is. Everything runs on the current stream; lengths and widths
are read on the device only. csrc/tree.hip has the kernels."""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from .kvcache import KVCache, check_table, refuse_gradients
from .lib import Entry, Lib, float32

WIDEST = 64  # tokens of a tree: the bits of a mask
DTYPES = {torch.bfloat16: 1, torch.float16: 2}


@functools.lru_cache(maxsize=None)
def _entries() -> tuple[Entry, Entry]:
    return Entry(name="ng_tree_attention", types="pqqqippppqiipqipppiiiiifppp"), Entry(name="ng_tree_mask", types="piip")


@functools.lru_cache(maxsize=1024)
def _work(B: int, T: int, H: int, G: int, dim: int, code: int, capacity: int) -> int:
    n = Lib().size("ng_tree_attention_work", B, T, H, G, dim, code, capacity)
    if n < 0:
        raise ValueError(f"{B} sequences of {T} tokens, {H} heads x {G}, dim {dim}, tables of {capacity} tokens: out of "
                         "range (tables hold at most 2^30 tokens)")
    return n


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """int64 [B, T]: bit j of [b, i] is set where token j is i or an ancestor of it. parents int32 [B, T], T <= 64: each
    token's parent, an earlier token; negative (or not earlier): the last cached token."""
    if parents.dtype != torch.int32 or parents.dim() != 2 or not 1 <= parents.shape[1] <= WIDEST or not parents.is_cuda:
        raise ValueError(f"parents must be int32 [B, 1 to {WIDEST}] on the GPU: got {tuple(parents.shape)} "
                         f"{parents.dtype} on {parents.device}")
    parents = parents.contiguous()
    out = torch.empty(parents.shape, dtype=torch.int64, device=parents.device)
    _entries()[1](parents.get_device(), parents.data_ptr(), *parents.shape, out.data_ptr())
    return out


def _check(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, cache: KVCache) -> torch.Tensor:
    if t.dtype != dtype or t.shape != shape or t.get_device() != cache.device:
        raise ValueError(f"{name} must be {dtype} {shape} on {cache.k.device}: got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.contiguous()


def tree_attention(q: torch.Tensor, cache: KVCache, table: torch.Tensor, lengths: torch.Tensor,
                   mask: torch.Tensor | None = None, widths: torch.Tensor | None = None, scale: float | None = None,
                   return_lse: bool = False):
    """Attention of q [B, T, heads * group, dim] (bfloat16 or float16, a 16-bit cache's own type; any strides over the
    first three) over the cached tokens and the tree; query head h reads the cache's head h // group.

    table    int32 [B, width]: the sequences' pages in order; keys whose entry is no page of the cache are masked
    lengths  int32 [B]: the cached tokens before the tree (held to 0 .. what the table covers)
    mask     int64 [B, T]: bit j of [b, i] lets tree token i see tree token j; None: a chain (i sees 0 .. i)
    widths   int32 [B]: the tree tokens in use (None: all T); the rows past them are zeros, whatever q holds there, their
             keys masked
    scale    the scores' factor, 1 / sqrt(dim) by default

    Returns the output in q's shape and type, and with return_lse the float32 [B, T, heads * group] logarithms of the
    softmax sums. A row that sees nothing is zeros, its logarithm -inf."""
    size, dtype = q.shape, q.dtype
    if len(size) != 4 or dtype not in DTYPES:
        raise ValueError(f"q must be [B, T, heads, dim] in bfloat16 or float16: got {tuple(size)} {dtype}")
    B, T, heads, dim = size
    if dim != cache.dim or heads < 1 or heads % cache.heads or not 1 <= T <= WIDEST:
        raise ValueError(f"q {tuple(size)} does not go with {cache.heads} cached heads of {cache.dim}: a multiple of the "
                         f"heads, 1 to {WIDEST} tokens")
    if cache.code >= 2 and dtype != cache.k.dtype:
        raise ValueError(f"a {cache.k.dtype} cache takes queries of its own type: got {dtype}")
    if q.get_device() != cache.device:
        raise ValueError(f"q is on {q.device}, the cache on {cache.k.device}")
    if q.requires_grad or forward_ad._current_level >= 0:
        refuse_gradients("tree_attention", q)
    check_table(cache, table)
    tables, width = table.shape
    if tables != B:
        raise ValueError(f"{tables} page tables for {B} sequences")
    lengths = _check("lengths", lengths, (B,), torch.int32, cache)
    if mask is not None:
        mask = _check("mask", mask, (B, T), torch.int64, cache)
    if widths is not None:
        widths = _check("widths", widths, (B,), torch.int32, cache)
    scale = 1 / math.sqrt(dim) if scale is None else float32("scale", scale)
    qb, qt, qh, qd = q.stride()
    if qd != 1 and dim > 1:
        q = q.contiguous()
        qb, qt, qh, _ = q.stride()
    device, group = cache.k.device, heads // cache.heads
    out = torch.empty(size, dtype=dtype, device=device)
    lse = torch.empty(size[:3], dtype=torch.float32, device=device) if return_lse else None
    work = torch.empty(_work(B, T, cache.heads, group, dim, cache.code, width * cache.page), dtype=torch.uint8, device=device)
    k, v, ks, vs = cache.addresses()
    _entries()[0](cache.device, q.data_ptr(), qb, qt, qh, DTYPES[dtype], k, v, ks, vs, cache.pages, cache.page, cache.code,
                  table.data_ptr(), table.stride(0), width, lengths.data_ptr(),
                  None if widths is None else widths.data_ptr(), None if mask is None else mask.data_ptr(), B, T,
                  cache.heads, group, dim, scale, out.data_ptr(), None if lse is None else lse.data_ptr(), work.data_ptr())
    return (out, lse) if return_lse else out
