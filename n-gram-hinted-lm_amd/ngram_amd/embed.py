"""Hint rows embedded, and the table's gradient: what a model does with the rows this package makes (the contract is the
reference's old_records/hint_runtime.py:381-418, the candidate mean: a position's candidates' embedding rows weighted by
its row's weights, summed over its slots, zero where a slot has no cell).

  embed(weight, tokens, weights=None, cell=None, scale=1.0)
      out[n] = scale * sum over the slots s with cell[n, s] > 0 and the entries e with weights[n, s, e] != 0 of
               weights[n, s, e] * weight[tokens[n, s, e]]
      without weights a lookup: out = scale * weight[tokens]
  HintEmbedding(vocab, dim, ...)   a module that holds the table; forward takes HintRows

Entries that do not count are not read. A counted token outside the table makes its position's output NaN (and adds to no
gradient): an IndexError would cost a device synchronization a call.

Differentiable in weight and weights. The table's gradient is dense and the same on every run: entries are sorted by token
(this library's stable radix sort) and each token's terms are added in order, in 32 bits, rounded once. Everything runs on
the current stream; csrc/embed.hip has the kernels."""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from .lib import Lib, i32

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TOKENS = {torch.int64: 8, torch.int32: 4, torch.uint16: 2}
_CELLS = {torch.int64: 8, torch.int32: 4, torch.int16: 2}


@functools.lru_cache(maxsize=None)
def _lib() -> Lib:
    return Lib()


@functools.lru_cache(maxsize=256)
def _grad_work(entries: int, vocab: int, dim: int) -> int:
    return _lib().size("ng_embed_grad_work", entries, vocab, dim)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension in memory order (a gradient may come expanded)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _Plan:
    """The checked arguments of one call: positions n, entries a position m, entries a slot, the leading shape."""

    def __init__(self, weight, tokens, weights, cell, scale):
        if weight.dim() != 2 or weight.dtype not in DTYPES:
            raise ValueError(f"weight must be [vocab, dim] in float32, bfloat16 or float16: got {tuple(weight.shape)} "
                             f"{weight.dtype}")
        if weight.shape[0] < 1 or weight.shape[1] < 1 or (weight.stride(1) != 1 and weight.shape[1] > 1):
            raise ValueError("weight's rows must be non-empty and contiguous")
        if tokens.dtype not in _TOKENS:
            raise ValueError(f"tokens must be int64, int32 or uint16: got {tokens.dtype}")
        if not weight.is_cuda:
            raise ValueError("embed runs on the GPU: weight is a CPU tensor")
        for name, t in (("tokens", tokens), ("weights", weights), ("cell", cell)):
            if t is not None and t.device != weight.device:
                raise ValueError(f"{name} is on {t.device}, weight on {weight.device}")
        if not math.isfinite(scale):
            raise ValueError(f"scale must be finite: {scale}")
        if weights is None:
            if cell is not None:
                raise ValueError("cell goes with weights")
            self.lead, self.n, self.m, self.entries = tuple(tokens.shape), tokens.numel(), 1, 1
        else:
            if weights.shape != tokens.shape or tokens.dim() not in (2, 3) or weights.dtype != torch.float32:
                raise ValueError(f"tokens and float32 weights must both be [n, entries] or [n, slots, entries]: got "
                                 f"{tuple(tokens.shape)} and {tuple(weights.shape)} {weights.dtype}")
            if tokens.shape[1:].numel() < 1:
                raise ValueError("rows need at least one entry")
            if cell is not None and (cell.shape != tokens.shape[:-1] or cell.dtype not in _CELLS):
                raise ValueError(f"cell must be {tuple(tokens.shape[:-1])} in int64, int32 or int16: got "
                                 f"{tuple(cell.shape)} {cell.dtype}")
            self.lead, self.n = (tokens.shape[0],), tokens.shape[0]
            self.m, self.entries = tokens.shape[1:].numel(), tokens.shape[-1]
        self.vocab, self.dim = weight.shape
        if self.n * self.m >= (1 << 31) - 64 or self.vocab >= 1 << 31:
            raise ValueError(f"{self.n * self.m} entries over {self.vocab} rows: at most 2^31 - 64 and 2^31 - 1")
        self.dtype, self.scale = i32(DTYPES[weight.dtype]), ctypes.c_float(scale)
        self.tsize = i32(_TOKENS[tokens.dtype])
        self.csize = i32(0 if cell is None else _CELLS[cell.dtype])
        self.shape = i32(self.m), i32(self.entries)


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, weights, cell, plan):
        out = torch.empty((*plan.lead, plan.dim), dtype=weight.dtype, device=weight.device)
        with torch.cuda.device(weight.device):
            _lib()("ng_embed", weight, weight.stride(0), plan.vocab, i32(plan.dim), plan.dtype, tokens, plan.tsize,
                   weights, cell, plan.csize, plan.n, *plan.shape, plan.scale, out)
        ctx.plan = plan
        ctx.save_for_backward(weight if ctx.needs_input_grad[2] else None, tokens, weights, cell)
        ctx.like = weight.dtype, weight.device
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        weight, tokens, weights, cell = ctx.saved_tensors
        plan, (dtype, device) = ctx.plan, ctx.like
        up = _rows(up.reshape(plan.n, plan.dim))
        dweight = dweights = None
        with torch.cuda.device(device):
            if ctx.needs_input_grad[0]:
                dweight = torch.empty((plan.vocab, plan.dim), dtype=dtype, device=device)
                work = torch.empty(_grad_work(plan.n * plan.m, plan.vocab, plan.dim), dtype=torch.uint8, device=device)
                _lib()("ng_embed_grad", up, up.stride(0), plan.vocab, i32(plan.dim), plan.dtype, tokens, plan.tsize,
                       weights, cell, plan.csize, plan.n, *plan.shape, plan.scale, dweight, work)
            if ctx.needs_input_grad[2]:
                dweights = torch.empty(weights.shape, dtype=torch.float32, device=device)
                _lib()("ng_embed_weight_grad", weight, weight.stride(0), up, up.stride(0), plan.vocab, i32(plan.dim),
                       plan.dtype, tokens, plan.tsize, cell, plan.csize, plan.n, *plan.shape, plan.scale, dweights)
        return dweight, None, dweights, None, None


def embed(weight: torch.Tensor, tokens: torch.Tensor, weights: torch.Tensor | None = None,
          cell: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
    """Embedded rows [n, dim] of tokens and float32 weights [n, entries] or [n, slots, entries], cell [n] or [n, slots]
    (None: every slot counts), or without weights the scaled lookup [*tokens.shape, dim]; in weight's type."""
    plan = _Plan(weight, tokens, weights, cell, float(scale))
    return _Embed.apply(weight, tokens.contiguous(), None if weights is None else weights.contiguous(),
                        None if cell is None else cell.contiguous(), plan)


class HintEmbedding(torch.nn.Module):
    """An embedding table for hint rows: forward(rows) takes HintRows (hints.py) and returns [n, dim]."""

    def __init__(self, vocab: int, dim: int, scale: float = 1.0, dtype: torch.dtype = torch.float32,
                 device: torch.device | str = "cuda"):
        super().__init__()
        self.scale = float(scale)
        self.weight = torch.nn.Parameter(torch.randn((vocab, dim), dtype=torch.float32, device=device).to(dtype))

    def forward(self, rows) -> torch.Tensor:
        return embed(self.weight, rows.tokens, rows.weights, rows.cell, self.scale)
