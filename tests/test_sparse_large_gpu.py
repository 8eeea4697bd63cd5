"""GPU: attention over kept pages and pages' bounds for more sequences than one launch has room for (a launch's threads are fewer
than 2^32), and bounds after writes of any length."""

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.sparse import PageBounds, sparse_attention

pytestmark = pytest.mark.gpu


def _cache(pages, heads, dim, codes="fp16", page=16):
    g = torch.Generator(device="cuda").manual_seed(pages)
    cache = KVCache.empty(pages, page, heads, dim, codes)
    k, v = (torch.randn((pages * page, heads, dim), generator=g, device="cuda").half() for _ in range(2))
    cache.write(k, v, torch.arange(pages * page, device="cuda"))
    bounds = PageBounds(cache)
    bounds.update(torch.arange(pages, dtype=torch.int32, device="cuda")[:, None], torch.zeros(pages, dtype=torch.int32, device="cuda"), page)
    return cache, bounds


@pytest.mark.parametrize("B,T,H,width,keep", [((1 << 20) + 9, 1, 8, 2, 1), ((1 << 19) + 5, 2, 8, 3, 2), ((1 << 21) + 3, 1, 4, 1, 4)])
def test_attention_in_passes(gpu, B, T, H, width, keep):
    cache, bounds = _cache(12, H, 1)
    g = torch.Generator(device="cuda").manual_seed(B)
    q = torch.randn((B, T, H, 1), generator=g, device="cuda").half()
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    some = torch.cat([torch.arange(7), B - 7 + torch.arange(7), torch.tensor([B // 2])]).cuda()
    table[some] = torch.randint(0, 12, (15, width), generator=g, device="cuda").int()
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    lengths[some] = torch.randint(0, 16 * width - T, (15,), generator=g, device="cuda").int()
    got = sparse_attention(q, cache, bounds, table, lengths, keep, first=0, return_lse=True, return_pages=True)
    want = sparse_attention(q[some], cache, bounds, table[some], lengths[some], keep, first=0, return_lse=True, return_pages=True)
    assert all(torch.equal(a[some], b) for a, b in zip(got, want))
    others = torch.ones(B, dtype=torch.bool, device="cuda")
    others[some] = False
    assert not got[0][others].any() and (got[1][others] == -float("inf")).all()


def test_bounds_in_passes(gpu):
    """2^26 places of pages; the first and last sequences have some."""
    cache, bounds = _cache(64, 8, 64, "int8")
    want, width, B = bounds.bounds.clone(), 8, (1 << 20) + 77
    bounds.bounds.fill_(7)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[0], table[B // 2], table[-1], table[-2] = (torch.arange(16 * i, 16 * i + 8, dtype=torch.int32) for i in range(4))
    bounds.update(table, torch.zeros(B, dtype=torch.int32, device="cuda"), 8 * 16)
    done = torch.arange(64) % 16 < 8
    assert torch.equal(bounds.bounds[done], want[done]) and (bounds.bounds[~done] == 7).all()


@pytest.mark.parametrize("start,count", [(0, (1 << 30) - 1), (-3, (1 << 30) - 1), (5, (1 << 30) - 1), (37, 1 << 29), (0, 16 * 6), (-17, 40),
                                         (-(1 << 31), (1 << 30) - 1), ((1 << 31) - 1, (1 << 30) - 1)])
def test_bounds_after_writes_of_any_length(gpu, start, count):
    """Positions past the table, and before its beginning, are nobody's."""
    B, width = 9, 7
    cache, bounds = _cache(B * width, 8, 64, "int8")
    want = bounds.bounds.clone()
    bounds.bounds.fill_(7)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(1)).int().view(B, width).cuda()
    bounds.update(table, torch.full((B,), start, dtype=torch.int32, device="cuda"), count)
    done = [j for j in range(width) if start < (j + 1) * 16 <= start + count]
    at = table[:, done].long().reshape(-1)
    left = torch.ones(B * width, dtype=torch.bool, device="cuda")
    left[at] = False
    assert torch.equal(bounds.bounds[at], want[at]) and (bounds.bounds[left] == 7).all()
