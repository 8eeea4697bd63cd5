"""GPU: the model-side operators together, as a model that verifies drafts uses them: a step's drafted tokens and their
positions' hint rows embedded (embed, HintEmbedding), their keys and values written behind the cached ones (KVCache), every
path of the tree attended at once (tree_attention, tree_mask), and the accepted path's keys and values written again, in
order. The same tokens decoded one at a time over a second cache give the same outputs.

Tolerance: both sides hold the same codes. Each output is off from the exact one by at most 2^-8 of itself (bfloat16), the
weights' 2^-11 (2^-8 over a bfloat16 cache) and the scores' error (below 2^-12 here: scores below 2^6, (64 + 6) 2^-24 of their terms' sum) times the
largest value; the two differ by at most twice that."""

import os

import pytest
import torch

from ngram_amd import hints as H
from ngram_amd.embed import HintEmbedding, embed
from ngram_amd.kvcache import KVCache
from ngram_amd.tree import tree_attention, tree_mask

pytestmark = pytest.mark.gpu

HEADS, GROUP, DIM, WIDTH, PAGE = 2, 2, 64, 128, 16


class Layer:
    """One attention layer over token embeddings plus the hint rows of the tokens' positions."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.table = (torch.randn((H.VOCAB, WIDTH), generator=g) * 0.5).bfloat16().cuda()
        torch.manual_seed(seed)
        self.hints = HintEmbedding(H.VOCAB, WIDTH, scale=0.5, dtype=torch.bfloat16)
        self.project = (torch.randn((WIDTH, (HEADS * GROUP + 2 * HEADS) * DIM), generator=g) / WIDTH**0.5).bfloat16().cuda()

    def qkv(self, tokens, rows):
        """Each [n, heads, DIM], views of one projection's output."""
        x = embed(self.table, tokens) + self.hints(rows)
        y = (x.float() @ self.project.float()).bfloat16().view(len(tokens), HEADS * GROUP + 2 * HEADS, DIM)
        return y[:, :HEADS * GROUP], y[:, HEADS * GROUP:-HEADS], y[:, -HEADS:]


def _rows(rows, at):
    return H.HintRows(rows.cell[at], rows.tokens[at], rows.weights[at])


@torch.no_grad()
@pytest.mark.parametrize("codes", ["int8", "fp8", "bf16"])
def test_a_tree_step_and_the_same_tokens_one_by_one(gpu, codes):
    os.environ.pop("HINT_NGRAM", None)
    n, T = 75, 9  # the context, and a tree: a chain of 5, two siblings of its third token, a child of one, a second root
    parents = torch.tensor([[-1, 0, 1, 2, 3, 1, 1, 5, -1]], dtype=torch.int32).cuda()
    path = [0, 1, 5, 7]  # the tokens accepted
    layer = Layer(7)
    rows = H.Hints("fake").val_span(0, n + T)
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, H.VOCAB, (n + T,), generator=g).cuda()
    depth = [0, 1, 2, 3, 4, 2, 2, 3, 0]  # a drafted token's position is its depth behind the context: its row is that one's
    drafted_rows = _rows(rows, torch.tensor([n + d for d in depth]).cuda())

    def cache_of(pages):
        return KVCache.empty(pages, PAGE, HEADS, DIM, codes), torch.randperm(pages, generator=g).int().view(1, -1).cuda()

    def start(length):
        return torch.tensor([length], dtype=torch.int32).cuda()

    # the context, then the tree in one step
    cache, table = cache_of(8)
    _, k, v = layer.qkv(tokens[:n], _rows(rows, slice(0, n)))
    cache.write(k, v, cache.slots(table, start(0), n)[0])
    q, tk, tv = layer.qkv(tokens[n:], drafted_rows)
    slots = cache.slots(table, start(n), T)[0]
    cache.write(tk, tv, slots)
    out = tree_attention(q[None], cache, table, start(n), tree_mask(parents))[0]

    # the accepted path's tokens one at a time, over a cache of their own
    other, its_table = cache_of(8)
    other.write(k, v, other.slots(its_table, start(0), n)[0])
    top = float(max(v.float().abs().max(), tv.float().abs().max()))
    for i, t in enumerate(path):
        other.write(tk[t:t + 1], tv[t:t + 1], other.slots(its_table, start(n + i), 1)[0])
        one = tree_attention(q[None, t:t + 1], other, its_table, start(n + i))[0, 0]
        assert ((out[t].double() - one.double()).abs() <= 2 * (2.0**-8 * one.double().abs() + (2.0**-8 if codes == "bf16" else
                2.0**-11) * top + 2.0**-12 * top)).all()

    # the tree's accepted tokens in order behind the context; the next token then sees the same cache on both sides
    keep = torch.tensor(path).cuda()
    cache.write(tk[keep], tv[keep], slots[:len(path)])
    at = torch.arange(n + len(path)).cuda()
    a, b = (c.read(c.slots(t, start(0), len(at))[0]) for c, t in ((cache, table), (other, its_table)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    nq = q[None, :1]
    last = [tree_attention(nq, c, t, start(n + len(path) - 1)) for c, t in ((cache, table), (other, its_table))]
    assert torch.equal(*last)
