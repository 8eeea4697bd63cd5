"""GPU: pages copied, moved and given to more rows than one launch has room for (a launch's threads are fewer than 2^32)."""

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.pages import PagePool, copy_pages

pytestmark = pytest.mark.gpu


def _fill(cache, pages, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (cache.k, cache.v):
        x = t.view(torch.uint8)
        x[pages] = torch.randint(0, 255, (len(pages), *x.shape[1:]), generator=g, device="cuda", dtype=torch.uint8)
    for t in (cache.k_scale, cache.v_scale):
        t[pages] = torch.rand((len(pages), *t.shape[1:]), generator=g, device="cuda")


def _same(a, at, b, to):
    return all(torch.equal(x.view(torch.uint8)[at], y.view(torch.uint8)[to]) for x, y in
               ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)))


def test_copies_in_passes(gpu):
    a, b = KVCache.empty(40, 16, 2, 64, "int8"), KVCache.empty(50, 16, 2, 64, "int8")
    _fill(a, torch.arange(40, device="cuda"), 1)
    n = (1 << 24) + 999
    src = torch.randint(0, 40, (n,), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    dst = torch.full((n,), -1, device="cuda")
    at = torch.cat([torch.arange(25), n - 25 + torch.arange(25)]).cuda()  # in the first pass, and in the last
    dst[at] = torch.randperm(50, generator=torch.Generator().manual_seed(3)).cuda()
    copy_pages(a, b, src, dst)
    assert _same(a, src[at], b, dst[at])


def test_a_move_in_passes(gpu):
    pages = (1 << 24) + 321
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    a, b = (KVCache.empty(pages, 16, 1, 64, "int8") for _ in range(2))
    some = torch.tensor([0, 1, 99, 1 << 20, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, pages - 2, pages - 1]).cuda()
    _fill(a, some, 4)
    pool, into = PagePool(a), PagePool(b)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")
    table = table[table != 99][None]  # all but one are in use
    pool.hold(table)
    out = pool.move(table, into)
    assert torch.equal(out[0], torch.arange(pages - 1, dtype=torch.int32, device="cuda"))
    kept = some[some != 99]
    assert _same(a, kept, b, kept - (kept > 99).long())
    assert int(into.missing) == 0 and int(into.refs.sum()) == pages - 1


def test_room_in_passes(gpu):
    """Rows times heads past a launch: the slots and a copy of the last rows."""
    heads, S = 128, (1 << 18) + 5
    cache = KVCache.empty(60, 16, heads, 1, "int8")
    pool = PagePool(cache)
    _fill(cache, torch.arange(60, device="cuda"), 5)
    table = torch.full((S, 2), -1, dtype=torch.int32, device="cuda")
    lengths, counts = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(2))
    table[-2:, 0], lengths[-2:] = 30, 5
    counts[-20:], counts[:3] = 2, 1
    pool.hold(table)
    slots = pool.reserve(table, lengths, 2, counts)
    assert slots[:3, 0].tolist() == [0, 16, 32] and (slots[:3, 1] == -1).all() and (slots[3:-20] == -1).all()
    want = [[(3 + i) * 16, (3 + i) * 16 + 1] for i in range(18)] + [[30 * 16 + 5, 30 * 16 + 6], [21 * 16 + 5, 21 * 16 + 6]]
    assert slots[-20:].tolist() == want and int(pool.missing) == 0
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        assert torch.equal(t[21, :, :5], t[30, :, :5])
