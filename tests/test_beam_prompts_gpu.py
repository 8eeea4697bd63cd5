"""GPU: a beam search over several prompts with the decoding operators together: each prompt's search is its own."""

import math

import pytest
import torch

from test_beam_search_gpu import DIM, END, HEADS, PAGE, VOCAB, WIDTH, Model

from ngram_amd.beam import beam_step, reorder
from ngram_amd.embed import embed
from ngram_amd.kvcache import KVCache
from ngram_amd.pages import PagePool
from ngram_amd.sparse import PageBounds, sparse_attention

pytestmark = pytest.mark.gpu


@torch.no_grad()
def test_searches_of_different_prompts_differ(gpu):
    """Three prompts, one of them twice: the like ones' searches are alike, the others' are not."""
    W, steps, B = 4, 12, 4
    model = Model(5)
    g = torch.Generator().manual_seed(11)
    a, b, c = (torch.randint(0, VOCAB, (n,), generator=g).cuda() for n in (40, 3, 77))
    prompt = [a, b, a, c]
    S, width = B * W, (77 + steps) // PAGE + 2
    cache = KVCache.empty(S * width, PAGE, HEADS, DIM, "bf16")
    bounds = PageBounds(cache)
    pool = PagePool(cache, bounds)
    table, lengths = torch.full((S, width), -1, dtype=torch.int32).cuda(), torch.zeros(S, dtype=torch.int32).cuda()
    for i, tokens in enumerate(prompt):
        row = slice(i * W, i * W + 1)
        _, k, v = model.qkv(tokens)
        cache.write(k, v, pool.reserve(table[row], lengths[row], len(tokens))[0])
        bounds.update(table[row], lengths[row], len(tokens))
        lengths[row] += len(tokens)
    pool.fork(table, lengths, torch.arange(B).repeat_interleave(W).cuda() * W)
    tokens = torch.stack([p[-1] for p in prompt]).repeat_interleave(W)
    scores = torch.full((B, W), -math.inf).cuda()
    scores[:, 0] = 0
    state, trace = torch.zeros((S, WIDTH)).cuda(), []
    grown, finished = torch.zeros((B, W), dtype=torch.int64).cuda(), torch.zeros((B, W), dtype=torch.bool).cuda()
    for _ in range(steps):
        q, k, v = model.qkv(tokens)
        cache.write(k, v, pool.reserve(table, lengths, 1)[:, 0])
        bounds.update(table, lengths, 1)
        out = sparse_attention(q[:, None], cache, bounds, table, lengths, 4, last=2)[:, 0]
        lengths += 1
        state = state * 0.5 + embed(model.table, tokens).float()
        step = beam_step(model.logits(out, state).view(B, W, VOCAB), scores, grown, finished, end=END, alpha=0.6)
        scores, grown, finished = step.scores, step.lengths, step.finished
        pool.fork(table, lengths, step.parents.reshape(-1))
        state, tokens = reorder(state, step.parents), step.tokens.reshape(-1)
        trace.append(step.tokens)
    whole = [tuple(x.reshape(-1).tolist()) for x in torch.stack(trace, 1)]
    assert len({whole[0], whole[1], whole[3]}) == 3
