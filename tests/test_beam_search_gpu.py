"""GPU: the decoding operators together, as a beam search uses them: each step chooses the hypotheses' continuations (beam_step),
forks their page tables (PagePool.fork), makes room (reserve), writes the new tokens' keys and values (KVCache) and the bounds
of the pages they complete (PageBounds), attends over the kept pages (sparse_attention), and reorders a state (reorder). The
same search in which every hypothesis keeps pages of its own, copied whole at each step, gives the same tokens and scores,
bit for bit: both attend over the same codes in the same order."""

import pytest
import torch

from ngram_amd.beam import beam_step, reorder
from ngram_amd.embed import embed
from ngram_amd.kvcache import KVCache
from ngram_amd.pages import PagePool, copy_pages
from ngram_amd.sparse import PageBounds, sparse_attention

pytestmark = pytest.mark.gpu

VOCAB, WIDTH, HEADS, GROUP, DIM, PAGE, END = 997, 128, 2, 2, 64, 16, 5


class Model:
    """One attention layer over token embeddings, its output and a running state as logits."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randn((VOCAB, WIDTH), generator=g).bfloat16().cuda()
        self.project = (torch.randn((WIDTH, (HEADS * GROUP + 2 * HEADS) * DIM), generator=g) / WIDTH**0.5).cuda()
        self.head = (torch.randn((HEADS * GROUP * DIM, VOCAB), generator=g) / 3).cuda()

    def qkv(self, tokens):
        y = (embed(self.table, tokens).float() @ self.project).bfloat16().view(len(tokens), HEADS * GROUP + 2 * HEADS, DIM)
        return y[:, :HEADS * GROUP], y[:, HEADS * GROUP:-HEADS], y[:, -HEADS:]

    def logits(self, out, state):
        return out.flatten(1).float() @ self.head + state @ self.head[:WIDTH] * 0.1


@torch.no_grad()
@pytest.mark.parametrize("codes", ["int8", "fp8", "bf16"])
@pytest.mark.parametrize("keep", [4, 64])
def test_shared_pages_and_pages_of_their_own(gpu, codes, keep):
    B, W, steps = 3, 4, 24
    S, prompts = B * W, [75, 1, 130]
    width = (max(prompts) + steps) // PAGE + 2
    model = Model(3)
    g = torch.Generator().manual_seed(9)
    prompt = [torch.randint(0, VOCAB, (n,), generator=g).cuda() for n in prompts]

    def search(shared):
        cache = KVCache.empty(S * width, PAGE, HEADS, DIM, codes)
        bounds = PageBounds(cache)
        pool = PagePool(cache, bounds)
        table = torch.full((S, width), -1, dtype=torch.int32).cuda()
        lengths = torch.zeros(S, dtype=torch.int32).cuda()
        for b, tokens in enumerate(prompt):  # each prompt is cached once, by its first beam
            row = slice(b * W, b * W + 1)
            _, k, v = model.qkv(tokens)
            cache.write(k, v, pool.reserve(table[row], lengths[row], len(tokens))[0])
            bounds.update(table[row], lengths[row], len(tokens))
            lengths[row] += len(tokens)
        first = torch.arange(B).repeat_interleave(W).cuda() * W

        def fork(parents):
            if shared:
                pool.fork(table, lengths, parents)
                return
            old, was = table.clone(), lengths.clone()  # whole copies: pages of the rows' own in another cache, and back
            spare = KVCache.empty(S * width, PAGE, HEADS, DIM, codes)
            spare_bounds = PageBounds(spare)
            mine = torch.arange(S * width).cuda()
            src = old[parents].reshape(-1).long()
            copy_pages(cache, spare, src, mine, bounds, spare_bounds)
            pool.clear()
            table.copy_(torch.where(src >= 0, mine, -1).view(S, width))
            pool.hold(table)
            lengths.copy_(was[parents])
            copy_pages(spare, cache, mine, mine, spare_bounds, bounds)

        fork(first)
        state = torch.zeros((S, WIDTH)).cuda()
        tokens = torch.tensor([int(p[-1]) for p in prompt]).repeat_interleave(W).cuda()
        scores = torch.full((B, W), -float("inf")).cuda()
        scores[:, 0] = 0
        grown, finished = torch.zeros((B, W), dtype=torch.int64).cuda(), torch.zeros((B, W), dtype=torch.bool).cuda()
        trace, pages = [], []
        for _ in range(steps):
            q, k, v = model.qkv(tokens)
            cache.write(k, v, pool.reserve(table, lengths, 1)[:, 0])
            bounds.update(table, lengths, 1)
            out = sparse_attention(q[:, None], cache, bounds, table, lengths, keep, last=2)[:, 0]
            lengths += 1
            state = state * 0.5 + embed(model.table, tokens).float()
            step = beam_step(model.logits(out, state).view(B, W, VOCAB), scores, grown, finished, end=END, alpha=0.6)
            scores, grown, finished = step.scores, step.lengths, step.finished
            fork(step.parents.reshape(-1))
            state, tokens = reorder(state, step.parents), step.tokens.reshape(-1)
            trace.append((step, lengths.clone()))
            pages.append(int((pool.refs > 0).sum()))
        assert int(pool.missing) == 0
        return trace, pages

    (a, used), (b, whole) = search(True), search(False)
    for (x, xl), (y, yl) in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y)) and torch.equal(xl, yl)
    assert torch.isfinite(a[-1][0].scores).all() and len({tuple(t) for t in a[-1][0].tokens.tolist()}) >= 1
    assert used[-1] < whole[-1]
    kinds = torch.cat([x.parents.reshape(-1) % W for x, _ in a])
    assert (kinds > 0).any()  # beams do change places
