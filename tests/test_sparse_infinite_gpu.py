"""GPU: the choice of pages (ngram_amd.sparse) where a 16-bit cache's keys, and so its pages' bounds, are infinite."""

import math

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.sparse import PageBounds, sparse_attention

pytestmark = pytest.mark.gpu


def _score(q, lo, hi):
    """sum over the group and the elements of the larger of q lo and q hi, a zero of q counting nothing: [tokens, pages]."""
    q, lo, hi = q[:, None], lo[None, :, None], hi[None, :, None]  # [T, 1, G, D], [1, pages, 1, D]
    x = torch.where(q > 0, q * hi, torch.where(q < 0, q * lo, torch.where(q != q, q, 0 * torch.where(lo.isinf(), 0.0, lo))))
    return x.sum((2, 3))


@pytest.mark.parametrize("B,T,G,dim,pages", [(1, 1, 1, 64, 60), (1, 1, 3, 128, 60), (130, 1, 2, 64, 60), (2, 3, 2, 100, 60), (1, 4, 1, 256, 60),
                                             (1, 9, 1, 64, 60), (2, 40, 2, 192, 60), (1, 1, 1, 256, 1300)])
def test_scores_from_infinite_bounds(gpu, B, T, G, dim, pages):
    """16-bit keys can be infinite: a page's score is its definition's, whatever the signs of the queries."""
    g = torch.Generator().manual_seed(T + dim + pages)
    cache = KVCache.empty(pages + 9, 16, 1, dim, "bf16")
    x = torch.randn(((pages + 9) * 16, 1, dim), generator=g).bfloat16().cuda()
    cache.write(x, x, torch.arange((pages + 9) * 16).cuda())
    bounds = PageBounds(cache)
    table = torch.randperm(pages + 9, generator=g)[:pages + 3].int()[None].expand(B, -1).contiguous().cuda()
    bounds.update(table, torch.zeros(B, dtype=torch.int32).cuda(), 16 * (pages + 3))
    tab = table[0].long()
    lo, hi = (bounds.bounds[:, 0, i] for i in (0, 1))
    for i in range(1, pages - 5):  # one page in three untouched; up to three elements of the others
        for _ in range(i % 3):
            at = int(torch.randint(0, dim, (1,), generator=g))
            kind = int(torch.randint(0, 4, (1,), generator=g))
            if kind < 2:
                hi[tab[i], at] = math.inf
            if kind in (1, 2):
                lo[tab[i], at] = -math.inf
            if kind == 3 and i % 5 == 0:  # every key of the page
                lo[tab[i], at] = hi[tab[i], at] = -math.inf if i % 2 else math.inf
    q = torch.randn((B, T, G, dim), generator=g).abs().bfloat16()
    q[:, :, :, ::2] *= -1
    q[:, :, :, 1::4] = 0
    if T > 1:
        q[:, 1] *= -1
    q[:, -1, :, :5] = 0
    q = q.cuda()
    lengths = torch.full((B,), 16 * pages + 3, dtype=torch.int32).cuda()
    keep = 20
    got = sparse_attention(q, cache, bounds, table, lengths, keep, return_pages=True)[1][:, :, 0].tolist()
    b0, b1 = lo[tab, :dim].double(), hi[tab, :dim].double()
    seen = pages + 1
    for b in range(0, B, 43):
        score = _score(q[b].double(), b0, b1)
        score = torch.where(score.isnan(), math.inf, score).tolist(), score.isnan().tolist()
        for t in range(T):
            n = (16 * pages + 3 + t) // 16 + 1
            assert seen <= n <= pages + 3
            rest = sorted(range(1, n - 1), key=lambda j: (not score[1][t][j], -score[0][t][j], j))[:keep - 2]
            assert got[b][t] == sorted([0, n - 1, *rest]), (b, t)
