"""GPU: attention for a tree of drafted tokens over a paged cache (ngram_amd.tree) against the definition in float64 over
the values the cache holds: cache types, head sizes, groups of query heads, one token to 64, lengths at every edge of a page
and a tile, ragged and empty sequences, unused tree rows, rows that see nothing, NaN and infinities in masked places, strided
queries, long caches past 2^32 bytes, streams, and the refusals.

Tolerances. u: the unit roundoff of the output (bfloat16 2^-8, float16 2^-11); up that of the softmax weights P in the
product with the values (2^-11 over 8-bit caches, which run on float16 products; a 16-bit cache's own type). A score's error
d is at most (dim + 6) 2^-24 of scale * sum |q||k| (32-bit sums of exact products, then three 32-bit operations and the
exponential's 2^-22), and moves P by a factor within exp(d); the sums over n keys are held in 32 bits. P of an 8-bit cache
below 2^-22 of the row's largest is rounded to a multiple of 2^-32 of it. So an output is off by at most
  u |o| + (up + 2 (e^d - 1) + (n + 8) 2^-24 + n 2^-32 * 2^8) A,  A = sum P |v| over the row plus max |v| * n * 2^-24
and the logarithm of the sum by d + (n + 8) 2^-24 + 2^-22 |lse|."""

import math

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.tree import tree_attention, tree_mask

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
UP = {torch.int8: 2.0**-11, torch.float8_e4m3fn: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _parents(B, T, g):
    return (torch.rand((B, T), generator=g) * (torch.arange(T) + 1)).int() - 1


def _ancestors(parents):
    B, T = parents.shape
    m = torch.zeros((B, T, T), dtype=torch.bool)
    for i in range(T):
        m[:, i, i] = True
        for b in range(B):
            p = int(parents[b, i])
            if 0 <= p < i:
                m[b, i] |= m[b, p]
    return m


def _bits(m):
    T = m.shape[-1]
    w = torch.tensor([1 << j if j < 63 else -(1 << 63) for j in range(T)])
    return (m.long() * w).sum(-1)


def _make(seed, B, T, heads, group, dim, codes, dtype, lengths, page=16, spare=0):
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
    x = [(torch.randn((pages * page, heads, dim), generator=g) * s).to(dtype).cuda() for s in (1.0, 2.0)]
    cache.write(x[0], x[1], torch.arange(pages * page).cuda())
    q = (torch.randn((B, T, heads * group, dim), generator=g) * 2).to(dtype).cuda()
    return q, cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), g


def _values(cache, table, b, n):
    at = cache.slots(table[b:b + 1], torch.zeros(1, dtype=torch.int32).cuda(), n)[0]
    k, v = cache.read(at, torch.float32)  # 8 bits: code * scale, off by 2^-24 from the kernel's factors at most
    return k.double(), v.double(), at >= 0


def _check(got, q, cache, table, lengths, sees, widths=None, scale=None, lse=None):
    """sees [B, T, T] bool"""
    B, T, heads, dim = q.shape
    group = heads // cache.heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    assert got.shape == q.shape and got.dtype == q.dtype
    for b in range(B):
        n0 = int(lengths[b])
        w = T if widths is None else int(widths[b])
        assert not got[b, w:].any()
        if lse is not None:
            assert (lse[b, w:] == -math.inf).all()
        n = min(n0 + w, table.shape[1] * cache.page)
        if w == 0:
            continue
        if n == 0:
            continue
        k, v, there = _values(cache, table, b, n)
        see = torch.ones((w, n), dtype=torch.bool).cuda()
        see[:, n0:] = sees[b, :w, :n - n0].cuda()
        see &= there
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            a = (q[b, :w, h].double() @ kh.T) * scale
            a = a.masked_fill(~see, -math.inf)
            z = torch.logsumexp(a, 1, keepdim=True)
            p = torch.where(z > -math.inf, torch.exp(a - torch.where(z > -math.inf, z, 0.0)), 0.0)
            want = p @ vh
            d = (dim + 6) * 2.0**-24 * abs(scale) * float((q[b, :w, h].double().abs() @ kh.abs().T).max()) + 2.0**-22
            A = p @ vh.abs() + vh.abs().max() * n * 2.0**-24
            bound = U[q.dtype] * want.abs() + (UP[cache.k.dtype] + 2 * math.expm1(d) + (n + 8) * 2.0**-24
                                               + n * 2.0**-24) * A + 2.0**-25
            off = (got[b, :w, h].double() - want).abs()
            assert torch.isfinite(got[b, :w, h]).all()
            assert (off <= bound).all(), (b, h, float((off - bound).max()), float(off.max()))
            if lse is not None:
                zl = lse[b, :w, h].double()
                none = z[:, 0] == -math.inf
                assert (zl[none] == -math.inf).all()
                zb = d + (n + 8) * 2.0**-24 + 2.0**-22 * (z[~none, 0].abs() + 16)
                assert ((zl[~none] - z[~none, 0]).abs() <= zb).all()


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.bfloat16),
                                         ("fp8", torch.float16), ("bf16", torch.bfloat16), ("fp16", torch.float16)])
@pytest.mark.parametrize("T,heads,group,dim", [(1, 2, 1, 64), (1, 2, 4, 128), (16, 1, 1, 80), (5, 3, 3, 96), (33, 2, 1, 64),
                                               (16, 2, 4, 128), (64, 1, 1, 192), (7, 1, 8, 256), (64, 1, 2, 128), (2, 1, 5, 1)])
def test_shapes(gpu, codes, dtype, T, heads, group, dim):
    lengths = [0, 1, 130, 511, 77]
    q, cache, table, ln, g = _make(T + dim, 5, T, heads, group, dim, codes, dtype, lengths)
    m = _ancestors(_parents(5, T, g))
    out, lse = tree_attention(q, cache, table, ln, _bits(m).cuda(), return_lse=True)
    _check(out, q, cache, table, ln, m, lse=lse)


@pytest.mark.parametrize("page", [16, 32, 64, 4096])
@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp16", torch.float16)])
def test_lengths_at_the_edges(gpu, page, codes, dtype):
    """Every length around a page's, a wave's and a tile's end."""
    lengths = [0, 1, 7, 8, 15, 16, 17, 30, 31, 32, 33, 63, 64, 65, 124, 127, 128, 129, 252, 255, 256, 257, 383, 384, 385]
    q, cache, table, ln, _ = _make(page, len(lengths), 4, 1, 2, 64, codes, dtype, lengths, page=page)
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)  # no mask: a chain
    chain = torch.tril(torch.ones(4, 4, dtype=torch.bool)).expand(len(lengths), 4, 4)
    _check(out, q, cache, table, ln, chain, lse=lse)


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("bf16", torch.bfloat16)])
def test_one_token(gpu, codes, dtype):
    lengths = [0, 5, 64, 300, 1000, 2047]
    q, cache, table, ln, _ = _make(3, 6, 1, 4, 8, 128, codes, dtype, lengths, page=64)
    _check(tree_attention(q, cache, table, ln), q, cache, table, ln, torch.ones(6, 1, 1, dtype=torch.bool))


@pytest.mark.parametrize("B", [1, 2, 70, 300])
def test_batches(gpu, B):
    """Work laid end to end over more sequences than a wave has lanes, lengths from none to thousands."""
    g = torch.Generator().manual_seed(B)
    lengths = (torch.rand(B, generator=g) ** 6 * 3000).int().tolist()
    lengths[B // 2] = 2900
    q, cache, table, ln, g = _make(B, B, 3, 2, 2, 64, "fp8", torch.bfloat16, lengths, page=32)
    m = _ancestors(_parents(B, 3, g))
    out, lse = tree_attention(q, cache, table, ln, _bits(m).cuda(), return_lse=True)
    _check(out, q, cache, table, ln, m, lse=lse)


@pytest.mark.parametrize("codes,dtype,T,group", [("int8", torch.bfloat16, 64, 4), ("fp8", torch.float16, 16, 4),
                                                 ("bf16", torch.bfloat16, 8, 4)])
def test_long_contexts(gpu, codes, dtype, T, group):
    q, cache, table, ln, g = _make(9, 2, T, 1, group, 128, codes, dtype, [20001, 9000], page=64, spare=700)
    m = _ancestors(_parents(2, T, g))
    out, lse = tree_attention(q, cache, table, ln, _bits(m).cuda(), return_lse=True)
    _check(out, q, cache, table, ln, m, lse=lse)


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp8", torch.bfloat16), ("fp16", torch.float16)])
def test_unused_rows_and_rows_that_see_nothing(gpu, codes, dtype):
    lengths = [0, 0, 40, 131, 7]
    widths = [0, 3, 9, 1, 20]
    q, cache, table, ln, g = _make(5, 5, 20, 2, 2, 64, codes, dtype, lengths)
    m = torch.rand((5, 20, 20), generator=g) < 0.3  # any mask, not only ancestors'
    m[1, 1] = False
    wd = torch.tensor(widths, dtype=torch.int32).cuda()
    out, lse = tree_attention(q, cache, table, ln, _bits(m).cuda(), wd, return_lse=True)
    _check(out, q, cache, table, ln, m, widths, lse=lse)
    assert not out[0].any() and not out[1, 1].any() and (lse[1, 1] == -math.inf).all()
    high = torch.tensor([-4, 3, 9, 1, 99], dtype=torch.int32).cuda()  # held to 0 .. T
    assert torch.equal(tree_attention(q, cache, table, ln, _bits(m).cuda(), high), out)


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp8", torch.float16), ("bf16", torch.bfloat16),
                                         ("fp16", torch.float16)])
def test_nothing_of_a_masked_key_shows(gpu, codes, dtype):
    """NaN, infinities and codes of NaN behind the sequences' ends, in pages of nobody and in tree tokens that a row does
    not see; the rows that see such a token are not finite."""
    T, lengths = 12, [37, 128, 5]
    q, cache, table, ln, g = _make(11, 3, T, 2, 2, 64, codes, dtype, lengths, spare=2)
    m = _ancestors(_parents(3, T, g))
    want, wl = tree_attention(q, cache, table, ln, _bits(m).cuda(), return_lse=True)
    _check(want, q, cache, table, ln, m, lse=wl)
    mine = torch.zeros(cache.pages * cache.page, dtype=torch.bool)
    for b in range(3):
        mine[cache.slots(table[b:b + 1], torch.zeros(1, dtype=torch.int32).cuda(), lengths[b] + T)[0].cpu()] = True
    stale = (~mine).nonzero()[:, 0].cuda()
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        bits = c.view(torch.uint8 if c.element_size() == 1 else torch.int16)
        bits[stale // 16, :, stale % 16] = -1 if c.element_size() == 2 else 0x7F  # NaN (int8: 127)
        if s is not None:
            s[stale // 16, :, stale % 16] = float("nan")
    table2 = table.clone()
    table2[table2 < 0] = 1 << 30
    for t in (table, table2):
        got, gl = tree_attention(q, cache, t, ln, _bits(m).cuda(), return_lse=True)
        assert torch.equal(got, want) and torch.equal(gl, wl)
    # tree token 4 of every sequence: a key of NaN; then a value row with an infinity and a NaN
    at = cache.slots(table, ln + 4, 1)[:, 0]
    k, v = cache.read(at, dtype)
    see4 = m[:, :, 4].cuda()
    for side in (0, 1):
        x = [k.clone(), v.clone()]
        x[side][:, :, 3], x[side][:, :, 40] = float("inf"), float("nan")
        cache.write(x[0], x[1], at)
        got, gl = tree_attention(q, cache, table, ln, _bits(m).cuda(), return_lse=True)
        assert torch.equal(got[~see4], want[~see4]) and torch.equal(gl[~see4], wl[~see4])
        assert torch.isnan(got[see4]).any(-1).all()
        if side == 1 and cache.k_scale is None:  # only the touched dimensions
            rest = [d for d in range(64) if d not in (3, 40)]
            assert torch.isfinite(got[see4][..., rest]).all() and not torch.isfinite(got[see4][..., [3, 40]]).any()


def test_scales_of_every_size(gpu):
    """Tokens whose values are 2^-40 to 2^40 of each other's: the scale joins the exponent, so P does not leave float16."""
    q, cache, table, ln, g = _make(13, 2, 3, 1, 2, 64, "int8", torch.float16, [300, 41])
    n = cache.pages * cache.page
    k = torch.randn((n, 1, 64), generator=g)
    v = torch.randn((n, 1, 64), generator=g) * torch.exp2((torch.rand((n, 1, 1), generator=g) - 0.5) * 24 - 8)
    v[::7] = 0
    cache.write(k.cuda(), v.cuda(), torch.arange(n).cuda())
    chain = torch.tril(torch.ones(3, 3, dtype=torch.bool)).expand(2, 3, 3)
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _check(out, q, cache, table, ln, chain, lse=lse)


@pytest.mark.parametrize("size", [2.0**-30, 2.0**-8, 1.0, 2.0**6])
def test_queries_of_every_size(gpu, size):
    q, cache, table, ln, g = _make(15, 2, 3, 1, 2, 64, "int8", torch.bfloat16, [300, 41])
    q = (q.float() * size).bfloat16()
    chain = torch.tril(torch.ones(3, 3, dtype=torch.bool)).expand(2, 3, 3)
    out, lse = tree_attention(q, cache, table, ln, scale=0.125, return_lse=True)
    _check(out, q, cache, table, ln, chain, scale=0.125, lse=lse)
    out = tree_attention(q, cache, table, ln, scale=-0.0625)
    _check(out, q, cache, table, ln, chain, scale=-0.0625)


def test_strides(gpu):
    """Queries as a view of one projection's output, at an offset no wide load is aligned to; a table with a row stride."""
    q, cache, table, ln, g = _make(17, 3, 6, 2, 2, 72, "fp8", torch.bfloat16, [60, 3, 200])
    m = _ancestors(_parents(3, 6, g))
    bits = _bits(m).cuda()
    want = tree_attention(q, cache, table, ln, bits)
    _check(want, q, cache, table, ln, m)
    wide = torch.zeros((3, 6, 4 * 72 + 5), dtype=torch.bfloat16).cuda()
    wide[..., 3:-2] = q.reshape(3, 6, -1)
    other = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    dims = q.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    table2 = torch.cat([table, table], 1)[:, :table.shape[1]]
    for x in (wide[..., 3:-2].view(3, 6, 4, 72), other, dims):
        assert torch.equal(tree_attention(x, cache, table2, ln, bits), want)


def test_page_entries_that_are_no_page(gpu):
    """A missing page masks its keys; lengths past the table are held to it."""
    q, cache, table, ln, _ = _make(19, 2, 2, 1, 1, 64, "int8", torch.bfloat16, [100, 60])
    table[0, 2], table[1, 0] = -1, cache.pages
    chain = torch.tril(torch.ones(2, 2, dtype=torch.bool)).expand(2, 2, 2)
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _check(out, q, cache, table, ln, chain, lse=lse)
    far = torch.tensor([1 << 30, -5], dtype=torch.int32).cuda()
    held = torch.tensor([table.shape[1] * 16, 0], dtype=torch.int32).cuda()
    assert torch.equal(tree_attention(q, cache, table, far), tree_attention(q, cache, table, held))


def test_cache_past_32_bits(gpu):
    """Pages that lie past 2^32 bytes."""
    pages = (1 << 32) // (4096 * 64) + 5
    k = torch.empty((pages, 1, 4096, 64), dtype=torch.int8, device="cuda")
    s = torch.empty((pages, 1, 4096), dtype=torch.float32, device="cuda")
    cache = KVCache(k, k, s, s, dim=64)
    table = torch.tensor([[pages - 1, 2], [pages - 2, pages - 3]], dtype=torch.int32).cuda()
    ln = torch.tensor([5000, 4094], dtype=torch.int32).cuda()
    at = cache.slots(table, torch.zeros(2, dtype=torch.int32).cuda(), 8192).reshape(-1)
    x = torch.randn((16384, 1, 64)).cuda()
    cache.write(x, x, at)
    q = torch.randn((2, 4, 2, 64)).bfloat16().cuda()
    chain = torch.tril(torch.ones(4, 4, dtype=torch.bool)).expand(2, 4, 4)
    _check(tree_attention(q, cache, table, ln), q, cache, table, ln, chain)


def test_another_stream_and_no_sequences(gpu):
    q, cache, table, ln, _ = _make(21, 2, 2, 1, 1, 64, "int8", torch.bfloat16, [100, 900])
    want = tree_attention(q, cache, table, ln)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tree_attention(q * 1, cache, table, ln)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    assert tree_attention(q[:0], cache, table[:0], ln[:0]).shape == (0, 2, 1, 64)


def test_same_on_every_run(gpu):
    q, cache, table, ln, _ = _make(23, 3, 8, 2, 4, 128, "fp8", torch.bfloat16, [3000, 10, 700])
    want = tree_attention(q, cache, table, ln, return_lse=True)
    for _ in range(3):
        got = tree_attention(q, cache, table, ln, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("B,T", [(1, 1), (3, 64), (100, 17)])
def test_tree_mask(gpu, B, T):
    g = torch.Generator().manual_seed(T)
    p = _parents(B, T, g)
    assert torch.equal(tree_mask(p.cuda()).cpu(), _bits(_ancestors(p)))
    chain = (torch.arange(T, dtype=torch.int32) - 1).expand(B, T).contiguous()
    assert torch.equal(tree_mask(chain.cuda()).cpu(), _bits(_ancestors(chain)))
    late = torch.full((B, T), T, dtype=torch.int32)  # no earlier token: no parent
    assert torch.equal(tree_mask(late.cuda()).cpu(), _bits(_ancestors(late)))


def test_refusals(gpu):
    q, cache, table, ln, _ = _make(25, 2, 4, 2, 2, 64, "int8", torch.bfloat16, [10, 20])
    mask, wd = torch.zeros((2, 4), dtype=torch.int64).cuda(), ln.clone()
    b16 = KVCache.empty(2, 16, 2, 64, "bf16")
    big = torch.zeros((1, 1), dtype=torch.int32).cuda().expand(2, 1 << 27)
    for args in ((q.float(), cache, table, ln), (q[0], cache, table, ln), (q[..., :63], cache, table, ln),
                 (q[:, :, :3], cache, table, ln), (q.cpu(), cache, table, ln), (q.repeat(1, 17, 1, 1), cache, table, ln),
                 (q[:, :0], cache, table, ln), (q, cache, table.long(), ln), (q, cache, table[:1], ln),
                 (q, cache, table[:, :0], ln), (q, cache, table, ln.long()), (q, cache, table, ln[:1]),
                 (q, cache, table, ln.cpu()), (q, cache, table, ln, mask.int()), (q, cache, table, ln, mask[:, :3]),
                 (q, cache, table, ln, mask, wd.long()), (q, cache, table, ln, mask, wd, float("inf")),
                 (q.half(), b16, table, ln), (q, cache, big, ln)):
        with pytest.raises(ValueError):
            tree_attention(*args)
    for p in (torch.zeros((2, 65), dtype=torch.int32).cuda(), torch.zeros((2, 4)).cuda(), torch.zeros(4, dtype=torch.int32).cuda(),
              torch.zeros((2, 4), dtype=torch.int32)):
        with pytest.raises(ValueError):
            tree_mask(p)


def _rows(got, q, cache, table, lengths, sees, scale=None, lse=None, skip=()):
    """_check row by row (but those of skip, pairs of tree token and head), for rows whose sizes differ: every bound is the
    row's own. The weights over 8-bit caches are resolved, a key, to 2^-33 of the largest weighted value (max of p times the
    value row's largest element), or to 2^-97 times the largest code where a value row of scale below 2^-64 has the largest
    weight. A row whose scores' error passes 1 has to be the value of its largest score, which then has to lead by more than
    that error."""
    B, T, heads, dim = q.shape
    group = heads // cache.heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    for b in range(B):
        n0 = int(lengths[b])
        n = n0 + T
        k, v, _ = _values(cache, table, b, n)
        for t in range(T):
            see = torch.ones(n, dtype=torch.bool)
            see[n0:] = sees[b, t]
            for h in range(heads):
                if (t, h) in skip:
                    continue
                kh, vh = k[see, h // group], v[see, h // group]
                x = q[b, t, h].double()
                a = (kh @ x) * scale
                d = (dim + 6) * 2.0**-24 * abs(scale) * float((kh.abs() @ x.abs()).max()) + 2.0**-22
                z = torch.logsumexp(a, 0)
                if d < 1:
                    p = torch.exp(a - z)
                    e = math.expm1(d)
                else:
                    top = a.topk(2).values
                    assert top[0] - top[1] > 2 * d + 60, "the case: its row has no clear largest score"
                    p, e = torch.nn.functional.one_hot(a.argmax(), len(a)).double(), 0.0
                want, A = p @ vh, p @ vh.abs()
                fine = (p * vh.abs().amax(1)).max() * n * 2.0**-33 + n * 2.0**-88
                bound = U[q.dtype] * want.abs() + (UP[cache.k.dtype] + 2 * e + (n + 8) * 2.0**-24) * A + fine + (
                    2.0**-25 if q.dtype == torch.float16 else 2.0**-134)
                off = (got[b, t, h].double() - want).abs()
                assert torch.isfinite(got[b, t, h]).all(), (b, t, h)
                assert (off <= bound).all(), (b, t, h, float((off - bound).max()), float(off.max()), float(want.abs().max()))
                if lse is not None:
                    zb = d + (n + 8) * 2.0**-24 + 2.0**-22 * (abs(float(z)) + 16)
                    assert abs(float(lse[b, t, h]) - float(z)) <= zb, (b, t, h, float(lse[b, t, h]), float(z), zb)


def _chain(B, T):
    return torch.tril(torch.ones(T, T, dtype=torch.bool)).expand(B, T, T)


@pytest.mark.parametrize("codes,dtype", [("int8", torch.bfloat16), ("fp8", torch.bfloat16), ("int8", torch.float16),
                                         ("fp16", torch.float16)])
@pytest.mark.parametrize("T,group,dim", [(5, 3, 64), (20, 2, 128), (20, 4, 192)])
def test_unused_rows_may_hold_anything(gpu, codes, dtype, T, group, dim):
    """Rows at or past widths are never read: whatever they hold, the others' outputs are the same bit for bit."""
    q, cache, table, ln, g = _make(31, 3, T, 2, group, dim, codes, dtype, [0, 200, 37])
    widths = [T - 2, 3, T // 2]
    wd = torch.tensor(widths, dtype=torch.int32).cuda()
    want, wl = tree_attention(q, cache, table, ln, None, wd, return_lse=True)
    _check(want, q, cache, table, ln, _chain(3, T), widths, lse=wl)
    for x in (1e9, 3e38, float("inf"), float("nan")):
        y = q.clone()
        for b, w in enumerate(widths):
            y[b, w:] = min(x, torch.finfo(dtype).max) if math.isfinite(x) else x
        got, gl = tree_attention(y, cache, table, ln, None, wd, return_lse=True)
        assert torch.equal(got, want) and torch.equal(gl, wl), x


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("T,group,dim", [(5, 3, 64), (12, 4, 128), (9, 2, 192), (6, 1, 250)])
def test_rows_of_different_sizes(gpu, codes, T, group, dim):
    """Query rows 2^-60 to 2^100 of each other in one block of rows: each is as right as alone."""
    q, cache, table, ln, g = _make(33, 2, T, 2, group, dim, codes, torch.bfloat16, [200, 33])
    q[:, 1] *= 2.0**-60
    q[:, 2] *= 2.0**40
    q[:, 3, 0] *= 2.0**100
    q[:, 3, -1] *= 2.0**20
    q[:, 4, 1] = 0
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _rows(out, q, cache, table, ln, _chain(2, T), lse=lse)


@pytest.mark.parametrize("size", [2.0**-126, 2.0**-100, 2.0**100, 2.0**120])
def test_queries_of_extreme_sizes(gpu, size):
    """Queries near the type's ends with a scale that makes ordinary scores of them."""
    q, cache, table, ln, _ = _make(35, 2, 3, 1, 2, 64, "int8", torch.bfloat16, [300, 41])
    q = (q.double() * size).bfloat16()
    assert torch.isfinite(q).all()
    scale = min(0.125 / size, 2.0**127)
    out, lse = tree_attention(q, cache, table, ln, scale=scale, return_lse=True)
    _rows(out, q, cache, table, ln, _chain(2, 3), scale=scale, lse=lse)


def test_a_query_row_that_is_not_finite(gpu):
    """An infinity or a NaN in a used row makes that row NaN and no other."""
    q, cache, table, ln, _ = _make(37, 2, 5, 1, 2, 64, "int8", torch.bfloat16, [200, 33])
    for x in (float("inf"), float("nan")):
        y = q.clone()
        y[:, 2, 1, 7] = x
        got, lse = tree_attention(y, cache, table, ln, return_lse=True)
        assert torch.isnan(got[:, 2, 1]).all()
        _rows(got, y, cache, table, ln, _chain(2, 5), lse=lse, skip=[(2, 1)])


def _with_values(seed, codes, lengths, size, zeros, lead, T=2):
    """A cache of values about `size`, zero rows at the positions `zeros` of every sequence, whose keys score `lead` more
    than ordinary ones (every query is about one direction)."""
    q, cache, table, ln, g = _make(seed, len(lengths), T, 1, 2, 64, codes, torch.bfloat16, lengths)
    base = torch.randn(64, generator=g)
    q = (base + 0.1 * torch.randn(q.shape, generator=g)).bfloat16().cuda()
    n = cache.pages * cache.page
    k = 0.3 * torch.randn((n, 1, 64), generator=g)
    v = torch.randn((n, 1, 64), generator=g) * size
    at = cache.slots(table, torch.zeros(len(lengths), dtype=torch.int32).cuda(), max(lengths) + T).cpu()
    for b in range(len(lengths)):
        for p in zeros:
            if p < lengths[b] + T:
                k[at[b, p]] = base * (lead * 8 / float(base @ base))  # scale 1/8: score `lead` with base
                v[at[b, p]] = 0
    cache.write(k.cuda(), v.cuda(), torch.arange(n).cuda())
    return q, cache, table, ln


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, 1e-5, 2.0**-20, 2.0**-40])
@pytest.mark.parametrize("lead", [0.0, 12.0, 40.0])
def test_value_rows_of_zeros(gpu, codes, size, lead):
    """Value rows of zeros take part in the softmax's sum and leave the others' weights their bits: at an ordinary score and
    at one far above, first, in the middle, last, and in the tree."""
    for zeros in ([0], [150], [5, 130, 201, 299], [300]):
        q, cache, table, ln = _with_values(41, codes, [300, 1, 210], size, zeros, lead)
        out, lse = tree_attention(q, cache, table, ln, return_lse=True)
        _rows(out, q, cache, table, ln, _chain(3, 2), lse=lse)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_scales_of_zero_stand_for_zeros(gpu, codes):
    """A scale of 0 over codes that are not 0 (a cache from elsewhere): zeros, as read() has them."""
    q, cache, table, ln = _with_values(43, codes, [300, 5], 1.0, [], 0.0)
    cache.v_scale.view(-1)[::3] = 0
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _rows(out, q, cache, table, ln, _chain(2, 2), lse=lse)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("first", [1e-35, 1e-30, 1e-20, 1e-17])
@pytest.mark.parametrize("rest", [1.0, 1e-4])
def test_tiny_values_first(gpu, codes, first, rest):
    """A first tile of values whose scales' inverses are near the largest float, then ordinary ones; and nothing else."""
    q, cache, table, ln = _with_values(45, codes, [300, 100, 700], rest, [], 0.0)
    n = cache.pages * cache.page
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn((n, 1, 64), generator=g) for _ in range(2))
    v *= rest
    at = cache.slots(table, torch.zeros(3, dtype=torch.int32).cuda(), 128).cpu()
    for b in range(3):
        for s in at[b]:
            if s >= 0:
                v[s] *= first / rest
    cache.write(k.cuda(), v.cuda(), torch.arange(n).cuda())
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _rows(out, q, cache, table, ln, _chain(3, 2), lse=lse)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("zeros", [False, True])
def test_value_sizes_far_apart(gpu, codes, zeros):
    """Values 2^-40 to 2^40 of each other's, with and without rows of zeros."""
    q, cache, table, ln, g = _make(47, 2, 3, 1, 2, 64, codes, torch.bfloat16, [300, 41])
    n = cache.pages * cache.page
    k = torch.randn((n, 1, 64), generator=g)
    v = torch.randn((n, 1, 64), generator=g) * torch.exp2((torch.rand((n, 1, 1), generator=g) - 0.5) * 80)
    if zeros:
        v[::7] = 0
    cache.write(k.cuda(), v.cuda(), torch.arange(n).cuda())
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _rows(out, q, cache, table, ln, _chain(2, 3), lse=lse)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_with_one_large_channel(gpu, codes, dim):
    """Keys whose codes are 0 but for a channel that the query has nothing in and another of the smallest code: a score is
    one product, to the last bits of itself. One key a sequence, so its logarithm is the score."""
    B = 40
    g = torch.Generator().manual_seed(dim)
    cache = KVCache.empty(B, 16, 1, dim, codes)
    q = (torch.randn((B, 1, 1, dim), generator=g) * 1000).bfloat16()
    k = torch.zeros((B, 1, dim))
    for b in range(B):
        top = 127.0 if codes == "int8" else 448.0
        k[b, 0, b % dim], k[b, 0, (b + 5) % dim] = top, 1.0
        q[b, 0, 0, b % dim] = 0
    table = torch.arange(B, dtype=torch.int32).view(B, 1).cuda()
    cache.write(k.cuda(), k.cuda(), torch.arange(B).cuda() * 16)
    none = torch.zeros(B, dtype=torch.int32).cuda()
    q = q.cuda()
    out, lse = tree_attention(q, cache, table, none, scale=1.0, return_lse=True)
    _rows(out, q, cache, table, none, _chain(B, 1), scale=1.0, lse=lse)


@pytest.mark.parametrize("side", [0, 1])
def test_codes_of_nan_in_a_masked_token(gpu, side):
    """An fp8 code that is itself NaN (a cache from elsewhere) in a tree token: only the rows that see it are NaN."""
    T = 12
    q, cache, table, ln, g = _make(49, 3, T, 2, 2, 64, "fp8", torch.bfloat16, [37, 128, 5])
    m = _ancestors(_parents(3, T, g))
    bits = _bits(m).cuda()
    want, wl = tree_attention(q, cache, table, ln, bits, return_lse=True)
    at = cache.slots(table, ln + 4, 1)[:, 0]
    held = (cache.k, cache.v)[side].view(torch.uint8)
    held[at // 16, :, at % 16, 9] = 0x7F
    held[at // 16, :, at % 16, 33] = 0xFF
    got, gl = tree_attention(q, cache, table, ln, bits, return_lse=True)
    see = m[:, :, 4].cuda()
    assert torch.equal(got[~see], want[~see]) and torch.equal(gl[~see], wl[~see])
    if side == 0:
        assert torch.isnan(got[see]).all()
    else:
        assert torch.isnan(got[see][..., [9, 33]]).all()
        rest = [d for d in range(64) if d not in (9, 33)]
        assert torch.equal(got[see][..., rest], want[see][..., rest]) and torch.equal(gl, wl)


def test_gradients_are_refused(gpu):
    """There is no backward pass: queries that require gradients raise instead of losing them."""
    import torch.autograd.forward_ad as fw

    q, cache, table, ln, _ = _make(51, 2, 2, 1, 1, 64, "int8", torch.bfloat16, [10, 20])
    want = tree_attention(q, cache, table, ln)
    x = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient"):
        tree_attention(x, cache, table, ln)
    with torch.no_grad():
        assert torch.equal(tree_attention(x, cache, table, ln), want)
    with torch.inference_mode():
        assert torch.equal(tree_attention(x, cache, table, ln), want)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="gradient"):
            tree_attention(fw.make_dual(q, torch.ones_like(q)), cache, table, ln)
        assert torch.equal(tree_attention(q, cache, table, ln), want)


def test_scales_that_are_no_float32_are_refused(gpu):
    q, cache, table, ln, _ = _make(53, 2, 2, 1, 1, 64, "int8", torch.bfloat16, [10, 20])
    for scale in (1e39, -1e39, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            tree_attention(q, cache, table, ln, scale=scale)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_negative_scales(gpu, codes):
    """Scales below 0 (a cache from elsewhere), of values and keys: code * scale, as read() has them; an infinite one in a
    masked token shows nowhere else."""
    q, cache, table, ln = _with_values(55, codes, [300, 5, 40], 1.0, [], 0.0)
    cache.v_scale.view(-1)[::3] *= -1
    cache.k_scale.view(-1)[1::5] *= -1
    out, lse = tree_attention(q, cache, table, ln, return_lse=True)
    _rows(out, q, cache, table, ln, _chain(3, 2), lse=lse)
    at = cache.slots(table, ln + 1, 1)[:, 0]
    for x in (-float("inf"), float("inf")):
        cache.v_scale[at // 16, :, at % 16] = x  # the second token: the first does not see it
        got, gl = tree_attention(q, cache, table, ln, return_lse=True)
        assert torch.equal(got[:, 0], out[:, 0]) and torch.equal(gl[:, 0], lse[:, 0])
        assert torch.isnan(got[:, 1]).any(-1).all()
