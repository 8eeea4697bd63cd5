"""A beam search's step: the best continuations of a batch's hypotheses (beams), chosen from a model's logits, and the beams'
states put in the chosen order. Their cached keys and values are not moved: pages.py forks the beams' page tables.

  beam_step(logits, scores, lengths=None, finished=None, keep=None, end=None, pad=None, alpha=0.0) -> BeamStep
  reorder(states, parents)

A candidate of beam w and token v has total = scores[w] + logits[w, v] - log sum exp logits[w]; a finished beam has one, its
padding token at its own score. Candidates are ranked by total / max(length, 1)^alpha, length being that of the beam with the
token (a finished one's own); equal ranks go to the lower beam, then the larger logit, then the lower token. A logit of -inf
is no candidate, nor are those of a beam whose score is -inf (all beams but the first at a search's start) or NaN, or whose
logits hold a NaN or +inf. Where fewer than `keep` candidates are left, the lowest (beam, token) of the others follow with a
score of -inf.

Log-sums, totals and ranks are held in 64 bits, the exponentials in 32. Nothing here has a backward pass, and nothing
synchronizes; everything runs on the current stream. csrc/beam.hip has the kernels."""

from __future__ import annotations

import functools
import math
from typing import NamedTuple, Sequence

import torch
from torch.autograd import forward_ad

from .kvcache import DTYPES, refuse_gradients
from .lib import Entry, Lib

MOST = 128  # beams of a sequence, and candidates kept


class BeamStep(NamedTuple):
    """The chosen candidates of each sequence, best first: scores float32 [B, keep]; parents int64 [B, keep], the rows b * W + w
    of the beams they continue; tokens int64 [B, keep]; finished bool [B, keep] (None: no beam can finish); lengths int64
    [B, keep] (None where no lengths were given)."""

    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor
    finished: torch.Tensor | None
    lengths: torch.Tensor | None


@functools.lru_cache(maxsize=None)
def _entries() -> tuple[Entry, Entry]:
    return (Entry(name="ng_beam_step", types="pqqippipiiiiiifpppppp"), Entry(name="ng_gather_rows", types="pqqqpqp"))


@functools.lru_cache(maxsize=None)
def _step() -> Entry:
    return Entry(name="ng_beam_step_alpha64", types="pqqippipiiiiiidpppppp")


@functools.lru_cache(maxsize=1024)
def _work(B: int, W: int, V: int, K: int) -> int:
    n = Lib().size("ng_beam_work", B, W, V, K)
    if n < 0:
        raise ValueError(f"{B} sequences of {W} beams, {V} tokens, {K} kept: at most 2^24 sequences, {MOST} beams and {MOST} "
                         "kept, 2^25 tokens, kept * ceil(tokens / 8192) at most 16384, and B * W * ceil(tokens / 8192) below 2^31")
    return n


def _check(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: int) -> torch.Tensor:
    if t.dtype != dtype or t.shape != shape or t.get_device() != device:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on GPU {device}: got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.contiguous()


def beam_step(logits: torch.Tensor, scores: torch.Tensor, lengths: torch.Tensor | None = None,
              finished: torch.Tensor | None = None, keep: int | None = None, end: int | None = None, pad: int | None = None,
              alpha: float = 0.0) -> BeamStep:
    """The `keep` best candidates (W by default) of each of B sequences' W beams: at most 2^25 tokens, and keep * ceil(V / 8192)
    at most 16384 (every keep up to 128 over 2^20 tokens).

    logits    [B, W, V] in float32, bfloat16 or float16, any strides over sequences and beams
    scores    float32 [B, W]: the beams' scores so far
    lengths   int64 or int32 [B, W]: their tokens so far, which alpha needs
    finished  bool [B, W]: the beams that have ended (their logits are not read)
    end       the token that ends a beam; pad: the one that a finished beam goes on with (`end` by default)
    alpha     the length normalisation's exponent, 0 or more"""
    size, dtype = logits.shape, logits.dtype
    if len(size) != 3 or dtype not in DTYPES or not logits.is_cuda:
        raise ValueError(f"logits must be [B, W, V] in float32, bfloat16 or float16 on the GPU: got {tuple(size)} {dtype} on "
                         f"{logits.device}")
    B, W, V = size
    keep = W if keep is None else int(keep)
    if not 1 <= W <= MOST or not 1 <= keep <= MOST or V < 1 or keep > W * V:
        raise ValueError(f"{W} beams, {V} tokens, {keep} kept: 1 to {MOST} beams, 1 to {MOST} kept of at least as many tokens")
    work = _work(B, W, V, keep)
    for name, token in (("end", end), ("pad", pad)):
        if token is not None and not 0 <= token < V:
            raise ValueError(f"{name} must be a token below {V}: {token}")
    pad = end if pad is None else pad
    if finished is not None and pad is None:
        raise ValueError("finished beams go on with a padding token: give end or pad")
    alpha = float(alpha)
    if not 0 <= alpha < math.inf or (alpha and lengths is None):
        raise ValueError(f"alpha must be finite, 0 or more, and needs lengths: {alpha}")
    if logits.requires_grad or scores.requires_grad or forward_ad._current_level >= 0:
        refuse_gradients("beam_step", logits, scores)
    gpu = logits.get_device()
    scores = _check("scores", scores, (B, W), torch.float32, gpu)
    if lengths is not None:
        lengths = _check("lengths", lengths, (B, W), torch.int32 if lengths.dtype == torch.int32 else torch.int64, gpu)
    if finished is not None:
        finished = _check("finished", finished, (B, W), torch.bool, gpu)
    if logits.stride(2) != 1:
        logits = logits.resolve_neg().contiguous()
    device, shape = logits.device, (B, keep)
    out = torch.empty(shape, dtype=torch.float32, device=device)
    # (one tensor's parts: an allocation costs a call of this size more than a view)
    parents, tokens, *more = torch.empty((2 if lengths is None else 3, B, keep), dtype=torch.int64, device=device).unbind(0)
    grown = more[0] if more else None
    done = torch.empty(shape, dtype=torch.bool, device=device) if finished is not None or end is not None else None
    scratch = torch.empty(work, dtype=torch.uint8, device=device)
    _step()(gpu, logits.data_ptr(), logits.stride(0), logits.stride(1), DTYPES[dtype], scores.data_ptr(), _at(lengths),
            0 if lengths is None else lengths.element_size(), _at(finished), B, W, V, keep, -1 if end is None else end,
            -1 if pad is None else pad, alpha, out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), _at(done), _at(grown),
            scratch.data_ptr())
    return BeamStep(out, parents, tokens, done, grown)


def _at(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def reorder(states: torch.Tensor | Sequence[torch.Tensor], parents: torch.Tensor):
    """The rows `parents` (int64, any shape: BeamStep's) of one state or of each of several, in new tensors [rows of parents,
    ...]: zeros where a parent is no row. States are [rows, ...] of any type, a row's elements in memory order."""
    if isinstance(states, torch.Tensor):
        return _reordered(states, parents)
    return [_reordered(s, parents) for s in states]


def _reordered(state: torch.Tensor, parents: torch.Tensor) -> torch.Tensor:
    if state.dim() < 1 or not state.is_cuda:
        raise ValueError(f"states must be [rows, ...] on the GPU: got {tuple(state.shape)} on {state.device}")
    if parents.dtype != torch.int64 or parents.get_device() != state.get_device():
        raise ValueError(f"parents must be int64 on {state.device}: got {parents.dtype} on {parents.device}")
    if state.requires_grad or forward_ad._current_level >= 0:
        refuse_gradients("reorder", state)
    if state.is_conj() or state.is_neg():  # (a bit of the tensor: its memory holds other values)
        state = state.resolve_conj().resolve_neg()
    rows, rest, size = state.shape[0], state.shape[1:], state.element_size()
    row = rest.numel() * size
    if not state.is_contiguous() and rows and not state[0].is_contiguous():
        state = state.contiguous()
    parents = parents.contiguous()
    n = parents.numel()
    out = torch.empty((n, *rest), dtype=state.dtype, device=state.device)
    _entries()[1](state.get_device(), state.data_ptr(), state.stride(0) * size, rows, row, parents.data_ptr(), n, out.data_ptr())
    return out
