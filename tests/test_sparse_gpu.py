"""GPU: attention over the pages that a score keeps (ngram_amd.sparse), against the definition in float64 over the values the
cache holds: the pages' bounds, the choice of pages (compared exactly: scores are 64-bit sums of exact products on both
sides), the attention over them; cache types, head sizes and groups, lengths and pages at every edge, ragged and unused rows,
masked places, strides, long caches, streams, graphs, and the refusals.

Tolerances are tree attention's (the same kernel over the kept pages): u the unit roundoff of the output (bfloat16 2^-8,
float16 2^-11), up that of the softmax weights P in the product with the values (2^-11 over 8-bit caches; a 16-bit cache's own
type), d a score's error, (dim + 6) 2^-24 of scale * sum |q||k| + 2^-22; over n keys an output is off by at most
  u |o| + (up + 2 (e^d - 1) + (n + 8) 2^-24 + n 2^-24) A + 2^-25,  A = sum P |v| over the row plus max |v| n 2^-24
and the logarithm of the sum by d + (n + 8) 2^-24 + 2^-22 (|lse| + 16). Bounds are exact."""

import math

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.sparse import PageBounds, sparse_attention
from ngram_amd.tree import tree_attention

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
UP = {torch.int8: 2.0**-11, torch.float8_e4m3fn: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _outward(lo, hi):
    """float32 to bfloat16, down and up."""
    def cut(x, up):
        near = x.bfloat16()
        wrong = near.float() < x if up else near.float() > x
        step = torch.where((near.float() > 0) == up, 1, -1).to(torch.int16)  # the next one up (down) in its bits
        out = torch.where(wrong, (near.view(torch.int16) + step).view(torch.bfloat16), near)
        tiny = torch.tensor([1 if up else -32767], dtype=torch.int16, device=x.device).view(torch.bfloat16)
        return torch.where(wrong & (near == 0), tiny, out)

    return torch.stack([cut(lo, False), cut(hi, True)], -2)


def _page_values(cache, page, count=None):
    at = page * cache.page + torch.arange(cache.page if count is None else count).cuda()
    return cache.read(at, torch.float32)  # [rows, heads, dim]


def _make(seed, B, T, heads, group, dim, codes, dtype, lengths, page=16, spare=0, apart=0.7):
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + T) // page) for n in lengths]
    width = max(need) + spare
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cache = KVCache.empty(pages, page, heads, dim, codes)
    k = torch.randn((pages, page, heads, dim), generator=g) + apart * torch.randn((pages, 1, heads, dim), generator=g)
    v = torch.randn((pages * page, heads, dim), generator=g) * 2
    cache.write(k.view(-1, heads, dim).to(dtype).cuda(), v.to(dtype).cuda(), torch.arange(pages * page).cuda())
    bounds = PageBounds(cache)
    every = torch.arange(pages, dtype=torch.int32)[:, None].cuda()
    bounds.update(every, torch.zeros(pages, dtype=torch.int32).cuda(), page)
    q = (torch.randn((B, T, heads * group, dim), generator=g) * 2).to(dtype).cuda()
    return q, cache, bounds, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()


def _check(q, cache, bounds, table, lengths, keep, widths=None, first=1, last=1, scale=None):
    out, lse, pages = sparse_attention(q, cache, bounds, table, lengths, keep, widths, first, last, scale, True, True)
    B, T, heads, dim = q.shape
    H, P, width = cache.heads, cache.page, table.shape[1]
    G = heads // H
    cap = width * P
    scale = 1 / math.sqrt(dim) if scale is None else scale
    assert out.shape == q.shape and out.dtype == q.dtype and pages.shape == (B, T, H, keep) and pages.dtype == torch.int32
    for b in range(B):
        n0 = min(max(int(lengths[b]), 0), cap)
        w = T if widths is None else min(max(int(widths[b]), 0), T)
        assert not out[b, w:].any() and (lse[b, w:] == -math.inf).all() and (pages[b, w:] == -1).all()
        if w == 0:
            continue
        tab = table[b].long()
        there = (tab >= 0) & (tab < cache.pages)
        at = torch.where(there, tab, 0)
        lo, hi = (bounds.bounds[at, :, i, :dim].double() for i in (0, 1))  # [width, H, dim]
        slots = (at[:, None] * P + torch.arange(P).cuda()).reshape(-1)
        k, v = (x.double() for x in cache.read(slots, torch.float32))  # [width * P, H, dim]
        for h in range(H):
            qh = q[b, :w, h * G:(h + 1) * G].double()  # [w, G, dim]
            score = qh.clamp(min=0).sum(1) @ hi[:, h].T + qh.clamp(max=0).sum(1) @ lo[:, h].T  # [w, width]
            score = torch.where(there, score, -math.inf).tolist()
            for t in range(w):
                keys = min(n0 + t + 1, cap)
                m = -(-keys // P)
                must = [j for j in range(m) if j < first or j >= m - last]
                rest = sorted((j for j in range(m) if first <= j < m - last), key=lambda j: (-score[t][j], j))
                want = list(range(m)) if m <= keep else sorted(must + rest[:keep - len(must)])
                assert pages[b, t, h].tolist() == want + [-1] * (keep - len(want)), (b, t, h)
                pos = (torch.tensor(want)[:, None] * P + torch.arange(P)).reshape(-1)
                pos = pos[pos < keys].cuda()
                pos = pos[there[pos // P]]
                n = len(pos)
                a = (qh[t] @ k[pos, h].T) * scale
                z = torch.logsumexp(a, 1)
                mine, zl = out[b, t, h * G:(h + 1) * G].double(), lse[b, t, h * G:(h + 1) * G].double()
                if n == 0:
                    assert not mine.any() and (zl == -math.inf).all()
                    continue
                p = torch.exp(a - z[:, None])
                o = p @ v[pos, h]
                d = (dim + 6) * 2.0**-24 * abs(scale) * float((qh[t].abs() @ k[pos, h].abs().T).max()) + 2.0**-22
                A = p @ v[pos, h].abs() + v[pos, h].abs().max() * n * 2.0**-24
                bound = U[q.dtype] * o.abs() + (UP[cache.k.dtype] + 2 * math.expm1(d) + (2 * n + 8) * 2.0**-24) * A + 2.0**-25
                off = (mine - o).abs()
                assert (off <= bound).all(), (b, t, h, float((off - bound).max()))
                assert ((zl - z).abs() <= d + (n + 8) * 2.0**-24 + 2.0**-22 * (z.abs() + 16)).all()
    return out, lse, pages


CODES = [("int8", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16), ("fp8", torch.float16),
         ("bf16", torch.bfloat16), ("fp16", torch.float16)]


@pytest.mark.parametrize("codes,dtype", CODES)
@pytest.mark.parametrize("T,heads,group,dim", [(1, 2, 1, 64), (1, 2, 4, 128), (3, 1, 16, 80), (2, 3, 3, 96), (1, 1, 17, 64), (5, 1, 2, 192),
                                               (1, 1, 8, 256), (2, 1, 40, 128), (2, 1, 5, 1)])
def test_shapes(gpu, codes, dtype, T, heads, group, dim):
    lengths = [0, 1, 130, 511, 77]
    _check(*_make(T + dim, 5, T, heads, group, dim, codes, dtype, lengths), 6, first=1, last=2)


@pytest.mark.parametrize("page", [16, 64, 256, 4096])
@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp16", torch.float16)])
def test_lengths_at_the_edges(gpu, page, codes, dtype):
    lengths = [0, 1, page - 1, page, page + 1, 2 * page - 2, 3 * page - 1, 3 * page, 5 * page - 1, 5 * page, 127, 128, 129, 255, 256]
    _check(*_make(page, len(lengths), 2, 1, 2, 64, codes, dtype, lengths, page=page), 3)


@pytest.mark.parametrize("keep,first,last", [(1, 0, 1), (2, 0, 2), (4, 2, 2), (5, 0, 1), (5, 4, 1), (40, 1, 1), (41, 1, 1), (1024, 3, 9)])
def test_pages_always_kept(gpu, keep, first, last):
    _check(*_make(keep, 3, 2, 2, 2, 64, "int8", torch.bfloat16, [16 * 40 - 1, 333, 16 * 41]), keep, first=first, last=last)


@pytest.mark.parametrize("dim", [64, 100, 192, 250])
@pytest.mark.parametrize("B,T,n", [(2, 1, 300), (66, 1, 40), (2, 2, 300), (1, 4, 70), (1, 5, 300), (1, 17, 33)])
def test_scores_of_every_row_size(gpu, dim, B, T, n):
    """One token by vector operations, apart from the choice and with it; up to four and more on the matrix units."""
    _check(*_make(dim + T, B, T, 2, 3, dim, "fp8", torch.bfloat16, [16 * n - 7 * b % 50 for b in range(B)]), 7)


@pytest.mark.parametrize("n,keep", [(1024, 1000), (1025, 17), (1023, 64), (4096, 100), (4097, 33), (9000, 500), (32768, 7)])
def test_many_pages(gpu, n, keep):
    """Sequences of as many pages as a wave, four waves or a block hold scores of, and one more."""
    _check(*_make(n, 2, 1, 1, 2, 64, "fp8", torch.bfloat16, [16 * n - 5, 16 * n // 3]), keep, first=1, last=3)


@pytest.mark.parametrize("T,group", [(64, 1), (200, 3)])
def test_a_prompts_chunk(gpu, T, group):
    _check(*_make(T, 2, T, 1, group, 64, "bf16", torch.bfloat16, [700, 0], page=32), 8, last=2)


@pytest.mark.parametrize("B", [70, 300])
def test_batches(gpu, B):
    g = torch.Generator().manual_seed(B)
    lengths = (torch.rand(B, generator=g) ** 6 * 3000).int().tolist()
    lengths[B // 2] = 2900
    _check(*_make(B, B, 1, 2, 2, 64, "fp8", torch.bfloat16, lengths, page=32), 5)


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp8", torch.bfloat16), ("fp16", torch.float16)])
def test_unused_rows(gpu, codes, dtype):
    q, *rest = _make(5, 5, 6, 2, 2, 64, codes, dtype, [0, 0, 400, 131, 7])
    widths = torch.tensor([0, 3, 5, 1, 6], dtype=torch.int32).cuda()
    out, lse, pages = _check(q, *rest, 4, widths)
    for b, w in enumerate(widths.tolist()):
        q[b, w:] = math.nan
    wide = torch.tensor([-4, 3, 5, 1, 99], dtype=torch.int32).cuda()  # held to 0 .. T
    again = sparse_attention(q, *rest, 4, wide, return_lse=True, return_pages=True)
    assert all(torch.equal(x, y) for x, y in zip(again, (out, lse, pages)))


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp8", torch.float16), ("bf16", torch.bfloat16), ("fp16", torch.float16)])
def test_nothing_of_a_masked_key_shows(gpu, codes, dtype):
    """NaN behind the tokens' positions, in pages of nobody, and in those pages' bounds."""
    T, lengths = 3, [337, 128, 5]
    q, cache, bounds, table, ln = _make(11, 3, T, 2, 2, 64, codes, dtype, lengths, spare=2)
    want = _check(q, cache, bounds, table, ln, 6)
    mine = torch.zeros(cache.pages * cache.page, dtype=torch.bool)
    for b in range(3):
        mine[cache.slots(table[b:b + 1], torch.zeros(1, dtype=torch.int32).cuda(), lengths[b] + T)[0].cpu()] = True
    stale = (~mine).nonzero()[:, 0].cuda()
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        bits = c.view(torch.uint8 if c.element_size() == 1 else torch.int16)
        bits[stale // 16, :, stale % 16] = -1 if c.element_size() == 2 else 0x7F
        if s is not None:
            s[stale // 16, :, stale % 16] = math.nan
    for b in range(3):  # the incomplete pages' bounds are never read, nor those of pages of nobody
        bounds.bounds[table[b, (lengths[b] + T - 1) // 16].long()] = math.nan
    used = set(table[table >= 0].tolist())
    for p in range(cache.pages):
        if p not in used:
            bounds.bounds[p] = math.nan
    table2 = table.clone()
    table2[table2 < 0] = 1 << 30
    for t in (table, table2):
        got = sparse_attention(q, cache, bounds, t, ln, 6, return_lse=True, return_pages=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_page_entries_that_are_no_page(gpu):
    """Pages missing inside a sequence rank last and are masked; a sequence without any page is zeros."""
    q, cache, bounds, table, ln = _make(4, 4, 2, 2, 2, 64, "int8", torch.bfloat16, [300, 290, 310, 16])
    table[0, [0, 3, 4, 9]] = -1
    table[1, 2:] = cache.pages + 5
    table[2, :] = -1
    table[3, 1] = -9  # its token's own page
    out, lse, _ = _check(q, cache, bounds, table, ln, 17, first=2, last=2)
    assert not out[2].any()
    _check(q, cache, bounds, table, ln, 6, first=2, last=2)


def test_scores_that_are_not_finite(gpu):
    """A NaN score is kept first (its page's keys show), scores of +inf before the finite ones, -inf behind them; equal ones go
    to the lower page."""
    q, cache, bounds, table, ln = _make(2, 1, 1, 1, 1, 64, "bf16", torch.bfloat16, [16 * 30])
    q.fill_(1.0)
    hi = bounds.bounds[:, 0, 1]
    tab = table[0].long()
    hi[tab] = 1.0
    hi[tab[20]], hi[tab[22], 3], hi[tab[9], 5], hi[tab[12], 0] = 2.0, math.inf, math.nan, -math.inf

    def kept(keep):
        return sparse_attention(q, cache, bounds, table, ln, keep, return_pages=True)[1][0, 0, 0].tolist()

    assert kept(3) == [0, 9, 30] and kept(4) == [0, 9, 22, 30] and kept(5) == [0, 9, 20, 22, 30]
    assert kept(8) == [0, 1, 2, 3, 9, 20, 22, 30]
    assert kept(30) == [j for j in range(31) if j != 12]
    hi[tab] = 0.0
    hi[tab[::2]] = -0.0
    assert kept(7) == [0, 1, 2, 3, 4, 5, 30]
    q.fill_(math.nan)
    assert kept(4) == [0, 1, 2, 30] and sparse_attention(q, cache, bounds, table, ln, 4).isnan().all()


@pytest.mark.parametrize("codes,dtype", CODES)
@pytest.mark.parametrize("dim,page", [(64, 16), (100, 32), (192, 128), (256, 64), (1, 16), (130, 256), (33, 512)])
def test_bounds(gpu, codes, dtype, dim, page):
    """The smallest and largest of a page's values, outward; of the pages that the positions complete and no other."""
    g = torch.Generator().manual_seed(dim)
    heads, pages = 3, 14
    cache = KVCache.empty(pages, page, heads, dim, codes)
    x = torch.randn((pages * page, heads, dim), generator=g) * torch.exp(2 * torch.randn((pages * page, heads, 1), generator=g))
    x = x.clamp(-3e4, 3e4).to(dtype).cuda()
    cache.write(x, x, torch.arange(pages * page).cuda())
    start = torch.randn((pages, heads, 2, cache.k.shape[3]), generator=g).bfloat16().cuda()
    bounds = PageBounds(cache, start.clone())
    table = torch.tensor([[5, 2, 9, -1], [7, 0, 13, 20], [1, 3, 4, 6], [8, 8, 8, 8], [10, 11, 12, -1]], dtype=torch.int32).cuda()
    P = page
    #  row 0: pages 0, 1 end with the positions; 1: page 0 held already and 1 is complete; 2: nothing; 3: past the table; 4: all
    begin, count = [0, P, 3 * P, 4 * P - 1, -2], 2 * P - 1
    begin[0] = 1
    bounds.update(table, torch.tensor(begin, dtype=torch.int32).cuda(), count)
    done = set()
    for b, s in enumerate(begin):
        for j in range(4):
            if (j + 1) * P <= s + count and (j + 1) * P > s and 0 <= table[b, j] < pages:
                done.add(int(table[b, j]))
    assert {5, 2} <= done and 1 not in done
    for p in range(pages):
        if p not in done:
            assert torch.equal(bounds.bounds[p], start[p])
            continue
        v = _page_values(cache, torch.tensor(p).cuda())[0]
        want = _outward(v.amin(0), v.amax(0))
        assert torch.equal(bounds.bounds[p, :, :, :dim], want)
        assert not bounds.bounds[p, :, :, dim:].any()
        assert (bounds.bounds[p, :, 0, :dim].float() <= v.amin(0)).all() and (bounds.bounds[p, :, 1, :dim].float() >= v.amax(0)).all()


def test_bounds_of_values_that_are_not_finite(gpu):
    cache = KVCache.empty(3, 16, 1, 64, "bf16")
    x = torch.randn((48, 1, 64)).bfloat16().cuda()
    x[3, 0, 5], x[20, 0, 1], x[21, 0, 2] = math.nan, math.inf, -math.inf
    cache.write(x, x, torch.arange(48).cuda())
    bounds = PageBounds(cache)
    bounds.update(torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), 48)
    b = bounds.bounds[:, 0]
    assert b[0, :, 5].isnan().all() and b.isnan().sum() == 2
    assert b[1, 1, 1] == math.inf and b[1, 0, 2] == -math.inf and b.isinf().sum() == 2
    eight = KVCache.empty(1, 16, 1, 64, "int8")
    eight.write(x[:16], x[:16], torch.arange(16).cuda())  # a row that holds a NaN has scale NaN
    bounds = PageBounds(eight)
    bounds.update(torch.tensor([[0]], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), 16)
    assert bounds.bounds.isnan().all()


def test_a_score_bounds_its_pages_keys(gpu):
    """No key of a page has a larger sum of products with the group's queries than the page's score."""
    q, cache, bounds, table, ln = _make(6, 1, 1, 2, 4, 96, "fp8", torch.bfloat16, [16 * 50])
    for h in range(2):
        qs = q[0, 0, 4 * h:4 * h + 4].double()
        for j in range(50):
            p = int(table[0, j])
            lo, hi = (bounds.bounds[p, h, i, :96].double() for i in (0, 1))
            k = _page_values(cache, torch.tensor(p).cuda())[0][:, h].double()
            assert float(torch.maximum(qs * lo, qs * hi).sum()) >= float((qs @ k.T).max(1).values.sum()) - 1e-9


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("bf16", torch.bfloat16)])
def test_all_pages_kept_is_tree_attention(gpu, codes, dtype):
    q, cache, bounds, table, ln = _make(3, 4, 1, 4, 8, 128, codes, dtype, [5, 64, 1000, 2047], page=64)
    a, al, _ = _check(q, cache, bounds, table, ln, 64)
    b, bl = tree_attention(q, cache, table, ln, return_lse=True)
    assert ((a.double() - b.double()).abs() <= 2.0**-6 * b.double().abs() + 2.0**-7).all()
    assert ((al - bl).abs() <= 2.0**-16 * bl.abs() + 2.0**-16).all()


def test_strides(gpu):
    q, cache, bounds, table, ln = _make(8, 3, 4, 2, 3, 72, "int8", torch.bfloat16, [500, 333, 90])
    want = sparse_attention(q, cache, bounds, table, ln, 5, return_lse=True, return_pages=True)
    big = torch.full((3, 4, 6, 80), math.nan, dtype=q.dtype).cuda()
    big[..., 3:75] = q  # rows that start at odd places
    wide = torch.full((3, table.shape[1] + 7), 12345, dtype=torch.int32).cuda()
    wide[:, :-7] = table
    long = torch.stack([ln, ln + 9], 1)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    apart = torch.stack([q, q], -1)[..., 0]
    for x in (big[..., 3:75], turned, apart):
        got = sparse_attention(x, cache, bounds, wide[:, :-7], long[:, 0], 5, return_lse=True, return_pages=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_scale_and_lengths_past_the_table(gpu):
    q, cache, bounds, table, ln = _make(9, 3, 2, 1, 2, 64, "fp16", torch.float16, [200, 40, 7])
    _check(q, cache, bounds, table, ln, 4, scale=-0.3)
    _check(q, cache, bounds, table, ln, 4, scale=0.0)
    far = torch.tensor([2**31 - 1, -5, table.shape[1] * 16 - 1], dtype=torch.int32).cuda()
    _check(q, cache, bounds, table, far, 4)


def test_cache_past_32_bits(gpu):
    """Keys of more than 2^32 bytes, bounds of more than 2^31: pages from both ends."""
    page, heads, dim = 16, 8, 128
    pages = (1 << 32) // (page * heads * dim) + 1000
    cache = KVCache.empty(pages, page, heads, dim, "int8")
    bounds = PageBounds(cache)
    order = torch.cat([torch.arange(pages - 60, pages), torch.arange(60)]).int()
    order = order[torch.randperm(120, generator=torch.Generator().manual_seed(1))]
    table = order[None].cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((120 * 16, heads, dim), generator=g, device="cuda") + torch.randn((120, 1, heads, dim), generator=g, device="cuda").expand(120, 16, heads, dim).reshape(-1, heads, dim)
    slots = cache.slots(table, torch.zeros(1, dtype=torch.int32).cuda(), 1920)[0]
    cache.write(x, x, slots)
    bounds.update(table, torch.zeros(1, dtype=torch.int32).cuda(), 1920)
    q = (torch.randn((1, 1, heads * 2, dim), generator=g, device="cuda") * 2).bfloat16()
    _check(q, cache, bounds, table, torch.tensor([1900], dtype=torch.int32).cuda(), 9)


def test_more_scores_than_a_pass_holds(gpu):
    """Rows whose scores fill the workspace several times over are taken in passes."""
    T, n = 2100, 8192
    q, cache, bounds, table, ln = _make(7, 1, 1, 2, 1, 64, "int8", torch.bfloat16, [16 * n - 3000])
    q = (torch.randn((1, T, 2, 64), generator=torch.Generator().manual_seed(3)) * 2).bfloat16().cuda()
    out, lse, pages = sparse_attention(q, cache, bounds, table, ln, 5, return_lse=True, return_pages=True)
    for t in (0, 1, 1023, 2047, 2048, 2049, 2099):
        o, l, p = _check(q[:, t:t + 1], cache, bounds, table, ln + t, 5)
        assert torch.equal(p[0, 0], pages[0, t])
        assert ((o[0, 0].double() - out[0, t].double()).abs() <= 2.0**-6).all()


def test_captured_and_another_stream(gpu):
    q, cache, bounds, table, ln = _make(21, 6, 2, 2, 4, 128, "fp8", torch.bfloat16, [2000, 5, 900, 0, 77, 1500])

    def step():
        bounds.update(table, ln, 2)
        return sparse_attention(q, cache, bounds, table, ln, 8, last=2, return_lse=True, return_pages=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    g = torch.Generator().manual_seed(2)
    for i in range(4):
        if i:
            q.copy_((torch.randn(q.shape, generator=g) * 2).bfloat16())
            ln.sub_(1).clamp_(min=0)
        want = step()
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_same_on_every_run(gpu):
    args = _make(31, 8, 1, 4, 4, 128, "int8", torch.bfloat16, [16 * 300] * 8)
    want = sparse_attention(*args, 20, return_lse=True, return_pages=True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(sparse_attention(*args, 20, return_lse=True, return_pages=True), want))


def test_no_sequences(gpu):
    q, cache, bounds, table, ln = _make(1, 1, 1, 1, 1, 64, "int8", torch.bfloat16, [20])
    out, pages = sparse_attention(q[:0], cache, bounds, table[:0], ln[:0], 2, return_pages=True)
    assert out.shape == (0, 1, 1, 64) and pages.shape == (0, 1, 1, 2)
    bounds.update(table[:0], ln[:0], 3)
    bounds.update(table, ln, 0)


def test_refusals(gpu):
    q, cache, bounds, table, ln = _make(1, 2, 1, 2, 2, 64, "int8", torch.bfloat16, [20, 40])
    ok = (q, cache, bounds, table, ln)

    def refused(*args, **kw):
        with pytest.raises(ValueError):
            sparse_attention(*args, **kw)

    for keep, first, last in ((0, 0, 1), (1025, 1, 1), (2, 1, 2), (3, -1, 1), (3, 1, 0)):
        refused(*ok, keep, first=first, last=last)
    for bad in (q[0], q.float(), q[..., :63], q[:, :, :3], q[:, :0], q.cpu()):
        refused(bad, *ok[1:], 4)
    refused(q[:1], *ok[1:], 4)
    other = KVCache.empty(4, 16, 2, 64, "int8")
    refused(q, cache, PageBounds(other), table, ln, 4)
    for bad in (table.long(), table.cpu(), table[:, :0], table[:1]):
        refused(q, cache, bounds, bad, ln, 4)
    for bad in (ln.long(), ln[:1], ln.cpu()):
        refused(q, cache, bounds, table, bad, 4)
        refused(*ok, 4, widths=bad)
        with pytest.raises(ValueError):
            bounds.update(table, bad, 1)
    refused(*ok, 4, scale=math.inf)
    refused(q, cache, bounds, torch.zeros((2, 32769), dtype=torch.int32).cuda(), ln, 4)
    half = KVCache.empty(4, 16, 2, 64, "fp16")
    refused(q, half, PageBounds(half), table, ln, 4)
    for bad in (bounds.bounds.float(), bounds.bounds[:-1], bounds.bounds.cpu(), bounds.bounds.transpose(1, 2)):
        with pytest.raises(ValueError):
            PageBounds(cache, bad)
    for count in (-1, 1 << 30):
        with pytest.raises(ValueError):
            bounds.update(table, ln, count)
    with pytest.raises(RuntimeError, match="backward"):
        sparse_attention(q.clone().requires_grad_(True), *ok[1:], 4)
    with torch.no_grad():
        sparse_attention(q.clone().requires_grad_(True), *ok[1:], 4)
