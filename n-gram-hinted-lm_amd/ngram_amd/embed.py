"""Hint rows embedded, and the table's gradient: what a model does with the rows this package makes (the contract is the
reference's old_records/hint_runtime.py:381-418, the candidate mean: a position's candidates' embedding rows weighted by
its row's weights, summed over its slots, zero where a slot has no cell).

  embed(weight, tokens, weights=None, cell=None, scale=1.0)
      out[n] = scale * sum over the slots s with cell[n, s] > 0 and the entries e with weights[n, s, e] != 0 of
               weights[n, s, e] * weight[tokens[n, s, e]]
      without weights a lookup: out = scale * weight[tokens]
  HintEmbedding(vocab, dim, ...)   a module that holds the table; forward takes HintRows

Entries that do not count are not read by the output and the table's gradient. A counted token outside the table makes its
position's output NaN (and adds to no gradient): an IndexError would cost a device synchronization a call. The weights'
gradient is the slope at 0 too: where a slot has a cell it reads the rows of weight 0, and is 0 for such an entry whose token
is outside the table.

Differentiable in weight and weights, in reverse mode (a forward-mode tangent raises). The table's gradient is dense and the
same on every run: entries are sorted by token (stably, by radix) and each token's terms are added in a fixed order, in 32
bits, rounded once. Everything runs on the current stream; csrc/embed.hip has the kernels."""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from .lib import Entry, Lib, float32

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TOKENS = {torch.int64: 8, torch.int32: 4, torch.uint16: 2}
_CELLS = {torch.int64: 8, torch.int32: 4, torch.int16: 2}


@functools.lru_cache(maxsize=None)
def _entries() -> tuple[Entry, Entry, Entry]:
    return (Entry(name="ng_embed", types="pqqiipippiqiifp"), Entry(name="ng_embed_grad", types="pqqiipippiqiifpp"),
            Entry(name="ng_embed_slopes", types="pqpqqiipippiqiifp"))


@functools.lru_cache(maxsize=256)
def _grad_work(entries: int, vocab: int, dim: int) -> int:
    return Lib().size("ng_embed_grad_work", entries, vocab, dim)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension in memory order (a gradient may come expanded)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, weights, cell, shape, scale):
        ctx.save_for_backward(weight if ctx.needs_input_grad[2] else None, tokens, weights, cell)
        ctx.of = shape, scale, weight.shape, weight.dtype, weight.device
        return _forward(weight, tokens, weights, cell, shape, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        weight, tokens, weights, cell = ctx.saved_tensors
        (lead, n, m, entries), scale, (vocab, dim), dtype, device = ctx.of
        up = _rows(up.reshape(n, dim))
        dt, csize = DTYPES[dtype], 0 if cell is None else _CELLS[cell.dtype]
        tsize, at = _TOKENS[tokens.dtype], _at(cell)
        dweight = dweights = None
        if ctx.needs_input_grad[0]:
            dweight = torch.empty((vocab, dim), dtype=dtype, device=device)
            work = torch.empty(_grad_work(n * m, vocab, dim), dtype=torch.uint8, device=device)
            _entries()[1](device.index, up.data_ptr(), up.stride(0), vocab, dim, dt, tokens.data_ptr(), tsize, _at(weights),
                          at, csize, n, m, entries, scale, dweight.data_ptr(), work.data_ptr())
        if ctx.needs_input_grad[2]:
            dweights = torch.empty(weights.shape, dtype=torch.float32, device=device)
            _entries()[2](device.index, weight.data_ptr(), weight.stride(0), up.data_ptr(), up.stride(0), vocab, dim, dt,
                          tokens.data_ptr(), tsize, _at(weights), at, csize, n, m, entries, scale, dweights.data_ptr())
        return dweight, None, dweights, None, None, None


def _at(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _forward(weight, tokens, weights, cell, shape, scale):
    lead, n, m, entries = shape
    vocab, dim = weight.shape
    out = torch.empty((*lead, dim), dtype=weight.dtype, device=weight.device)
    _entries()[0](weight.get_device(), weight.data_ptr(), weight.stride(0), vocab, dim, DTYPES[weight.dtype],
                  tokens.data_ptr(), _TOKENS[tokens.dtype], _at(weights), _at(cell),
                  0 if cell is None else _CELLS[cell.dtype], n, m, entries, scale, out.data_ptr())
    return out


def _check(weight, tokens, weights, cell) -> tuple:
    """The shape of the call: the output's leading shape, positions, entries a position and entries a slot."""
    if weight.dim() != 2 or weight.dtype not in DTYPES:
        raise ValueError(f"weight must be [vocab, dim] in float32, bfloat16 or float16: got {tuple(weight.shape)} "
                         f"{weight.dtype}")
    vocab, dim = weight.shape
    if vocab < 1 or dim < 1 or (weight.stride(1) != 1 and dim > 1):
        raise ValueError("weight's rows must be non-empty and contiguous")
    if tokens.dtype not in _TOKENS:
        raise ValueError(f"tokens must be int64, int32 or uint16: got {tokens.dtype}")
    device = weight.get_device()
    if device < 0:
        raise ValueError("embed runs on the GPU: weight is a CPU tensor")
    for name, t in (("tokens", tokens), ("weights", weights), ("cell", cell)):
        if t is not None and t.get_device() != device:
            raise ValueError(f"{name} is on {t.device}, weight on {weight.device}")
    size = tokens.shape
    if weights is None:
        if cell is not None:
            raise ValueError("cell goes with weights")
        shape = size, tokens.numel(), 1, 1
    else:
        if weights.shape != size or len(size) not in (2, 3) or weights.dtype != torch.float32:
            raise ValueError(f"tokens and float32 weights must both be [n, entries] or [n, slots, entries]: got "
                             f"{tuple(size)} and {tuple(weights.shape)} {weights.dtype}")
        shape = size[:1], size[0], size[1:].numel(), size[-1]
        if shape[2] < 1:
            raise ValueError("rows need at least one entry")
        if cell is not None and (cell.shape != size[:-1] or cell.dtype not in _CELLS):
            raise ValueError(f"cell must be {tuple(size[:-1])} in int64, int32 or int16: got {tuple(cell.shape)} "
                             f"{cell.dtype}")
    if shape[1] * shape[2] >= (1 << 31) - 64 or vocab >= 1 << 31:
        raise ValueError(f"{shape[1] * shape[2]} entries over {vocab} rows: at most 2^31 - 65 and 2^31 - 1")
    return shape


def embed(weight: torch.Tensor, tokens: torch.Tensor, weights: torch.Tensor | None = None,
          cell: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
    """Embedded rows [n, dim] of tokens and float32 weights [n, entries] or [n, slots, entries], cell [n] or [n, slots]
    (None: every slot counts), or without weights the scaled lookup [*tokens.shape, dim]; in weight's type."""
    scale = float32("scale", scale)
    shape = _check(weight, tokens, weights, cell)
    tokens = tokens.contiguous()
    weights = None if weights is None else weights.contiguous()
    cell = None if cell is None else cell.contiguous()
    if (torch.is_grad_enabled() and (weight.requires_grad or (weights is not None and weights.requires_grad))
            or forward_ad._current_level >= 0):  # a level of forward mode is open: the function refuses tangents
        return _Embed.apply(weight, tokens, weights, cell, shape, scale)
    return _forward(weight, tokens, weights, cell, shape, scale)


class HintEmbedding(torch.nn.Module):
    """An embedding table for hint rows: forward(rows) takes HintRows (hints.py) and returns [n, dim]."""

    def __init__(self, vocab: int, dim: int, scale: float = 1.0, dtype: torch.dtype = torch.float32,
                 device: torch.device | str = "cuda"):
        super().__init__()
        self.scale = float(scale)
        self.weight = torch.nn.Parameter(torch.randn((vocab, dim), dtype=torch.float32, device=device).to(dtype))

    def forward(self, rows) -> torch.Tensor:
        return embed(self.weight, rows.tokens, rows.weights, rows.cell, self.scale)
