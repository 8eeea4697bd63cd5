"""GPU: who holds a cache's pages (ngram_amd.pages), against a pool kept in Python lists: forks, reservations, copies on a write,
exhaustion, moves, the pages' contents. Everything here is whole numbers or moved bytes: all comparisons are exact."""

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.pages import PagePool, copy_pages
from ngram_amd.sparse import PageBounds

pytestmark = pytest.mark.gpu


class Plain:
    """The pool's definition, a step at a time."""

    def __init__(self, pages, page, rows, width):
        self.pages, self.page, self.width = pages, page, width
        self.table = [[-1] * width for _ in range(rows)]
        self.length = [0] * rows
        self.missing = 0

    def refs(self):
        n = [0] * self.pages
        for r in self.table:
            for e in r:
                if 0 <= e < self.pages:
                    n[e] += 1
        return n

    def fork(self, parents):
        S = len(self.table)
        self.table = [list(self.table[p]) if 0 <= p < S else [-1] * self.width for p in parents]
        self.length = [self.length[p] if 0 <= p < S else 0 for p in parents]

    def reserve(self, count, counts=None):
        P = self.page
        refs = self.refs()
        free = [g for g in range(self.pages) if refs[g] == 0]
        own = [count if counts is None else max(0, min(count, c)) for c in counts or [count] * len(self.table)]
        spans = [range(n // P, min(self.width, (n + c - 1) // P + 1)) if c else range(0) for n, c in zip(self.length, own)]
        asking = {}
        for r, span in enumerate(spans):
            for c in span:
                if self.table[r][c] >= 0:
                    asking.setdefault(self.table[r][c], []).append((r, c))
        keeps = {x[0] for g, x in asking.items() if len(x) == refs[g]}
        copies, refused, at = [], set(), 0
        for r, span in enumerate(spans):
            for c in span:
                if (r, c) in keeps:
                    continue
                if at == len(free):
                    refused.add((r, c))
                    continue
                if self.table[r][c] >= 0 and self.length[r] > c * P:
                    copies.append((self.table[r][c], free[at], self.length[r] - c * P))
                self.table[r][c] = free[at]
                at += 1
        self.missing += len(refused)
        return [[-1 if i >= own[r] or x // P >= self.width or (r, x // P) in refused else self.table[r][x // P] * P + x % P
                 for i, x in enumerate(range(n, n + count))] for r, n in enumerate(self.length)]


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


class Both:
    """The pool and the plain one, side by side; every written token has a number, which its key and value hold."""

    def __init__(self, pages, page, rows, width, codes="bf16", heads=2, dim=5):
        self.plain = Plain(pages, page, rows, width)
        self.cache = KVCache.empty(pages, page, heads, dim, codes)
        self.pool = PagePool(self.cache)
        self.table = torch.full((rows, width), -1, dtype=torch.int32).cuda()
        self.lengths = torch.zeros(rows, dtype=torch.int32).cuda()
        self.history = [[] for _ in range(rows)]
        self.number = 0

    def check(self):
        p = self.plain
        assert self.table.tolist() == p.table
        assert self.lengths.tolist() == p.length
        assert self.pool.refs.tolist() == p.refs()
        assert int(self.pool.missing) == p.missing

    def fork(self, parents):
        self.pool.fork(self.table, self.lengths, _dev(parents, torch.int64))
        self.plain.fork(parents)
        S = len(self.history)
        self.history = [list(self.history[p]) if 0 <= p < S else [] for p in parents]
        self.check()

    def append(self, count, counts=None):
        slots = self.pool.reserve(self.table, self.lengths, count, None if counts is None else _dev(counts))
        want = self.plain.reserve(count, counts)
        assert slots.tolist() == want
        self.check()
        S = len(self.history)
        numbers = torch.arange(self.number, self.number + S * count).view(S, count) % 251  # exact in every type
        self.number += S * count
        x = numbers.reshape(-1, 1, 1).expand(-1, self.cache.heads, self.cache.dim).float() + 1
        x = x.to(self.cache.k.dtype if self.cache.code >= 2 else torch.float32).cuda()
        self.cache.write(x, -x, slots.reshape(-1))
        for s in range(S):
            n = sum(w >= 0 for w in want[s])
            assert all(w >= 0 for w in want[s][:n])
            self.history[s] += numbers[s, :n].tolist()
            self.plain.length[s] += n
        self.lengths.copy_(_dev(self.plain.length))
        self.read()

    def read(self):
        for s, h in enumerate(self.history):
            if not h:
                continue
            k, v = self.cache.read(self.cache.slots(self.table[s:s + 1], _dev([0]), len(h))[0], torch.float32)
            got = torch.stack([k, -v]) - 1
            want = torch.tensor(h).cuda().view(1, -1, 1, 1)
            assert ((got - want).abs() < 0.5).all()  # an 8-bit row is one number: its scale's rounding


@pytest.mark.parametrize("codes", ["int8", "fp8", "bf16", "fp16"])
@pytest.mark.parametrize("page,rows,count", [(16, 5, 1), (16, 8, 7), (32, 3, 40), (16, 70, 3), (64, 6, 64)])
def test_histories(gpu, codes, page, rows, count):
    """Forks and appended tokens in turn: every row reads back what its own past holds."""
    g = torch.Generator().manual_seed(page + rows)
    width = (11 * count + 200) // page + 1
    b = Both(rows * (width + 2), page, rows, width, codes)
    b.append(min(37, page * width), [1 + 5 * s % 37 for s in range(rows)])
    for step in range(6):
        kind = step % 3
        if kind == 0:
            parents = torch.randint(0, rows, (rows,), generator=g).tolist()  # some die, some have several children
        elif kind == 1:
            parents = torch.randperm(rows, generator=g).tolist()
        else:
            parents = [int(x) if x < rows else -1 for x in torch.randint(0, rows + 2, (rows,), generator=g)]
        b.fork(parents)
        b.append(count)
    b.fork([-1] * rows)
    assert not b.pool.refs.any() and not b.table.ge(0).any()


@pytest.mark.parametrize("codes", ["int8", "bf16"])
def test_many_requests(gpu, codes):
    """More requests in a call than a block's threads, for pages in common among them."""
    rows, g = 700, torch.Generator().manual_seed(8)
    b = Both(rows * 7, 16, rows, 6, codes, heads=1)
    b.append(20, [20 if s % 3 else 0 for s in range(rows)])
    for _ in range(2):
        b.fork(torch.randint(0, rows // 4, (rows,), generator=g).tolist())
        b.append(3)
    b.append(30, torch.randint(-5, 31, (rows,), generator=g).tolist())


def test_pages_run_out(gpu):
    """What was to be had goes to the first rows; the others' slots are -1 and nobody's rows are touched."""
    b = Both(7, 16, 4, 4)
    b.append(20, [20, 16, 3, 1])
    b.fork([0, 0, 0, 0])
    assert int(b.pool.missing) == 0
    b.append(5, [5, 5, 5, 5])  # a page each but one: 7 pages hold 2 + 3 copies
    b.append(40, [0, 40, 40, 40])
    assert int(b.pool.missing) > 0
    b.fork([1, 1, -1, 1])
    b.append(1)
    b.pool.clear()
    assert not b.pool.refs.any() and int(b.pool.missing) == 0


def test_shared_pages_ahead_of_the_length(gpu):
    """Reserved pages that hold no token yet are shared by a fork and left to one."""
    b = Both(40, 16, 3, 6)
    b.append(20, [20, 0, 0])
    slots = b.pool.reserve(b.table, b.lengths, 40)
    assert slots.tolist() == b.plain.reserve(40)
    b.check()
    b.fork([0, 0, 0])
    b.append(40)
    b.fork([2, 1, 0])
    # a length cut back into a shared page (drafts not accepted)
    b.fork([0, 0, 1])
    for s in range(3):
        del b.history[s][25:]
        b.plain.length[s] = 25
    b.lengths.fill_(25)
    b.append(3)


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 64, 5000, 32768, 32769, 100001])
def test_the_lowest_free_pages(gpu, pages):
    """Free bits at every edge of a word and a block's pass; all pages given, then a few let go and given again."""
    cache = KVCache.empty(pages, 16, 1, 1, "bf16")
    pool = PagePool(cache)
    table = torch.full((1, pages + 1), -1, dtype=torch.int32).cuda()
    lengths = torch.zeros(1, dtype=torch.int32).cuda()
    slots = pool.reserve(table, lengths, pages * 16)
    assert torch.equal(slots[0].cpu(), torch.arange(pages * 16)) and (pool.refs == 1).all() and int(pool.missing) == 0
    assert pool.reserve(table[:, pages:], lengths, 1).tolist() == [[-1]] and int(pool.missing) == 1
    g = torch.Generator().manual_seed(pages)
    gone = torch.randperm(pages, generator=g)[:min(pages, 40)].sort().values
    other = torch.full((1, 41), -1, dtype=torch.int32)
    other[0, :len(gone)] = gone.int()
    other = other.cuda()
    table[0, gone.cuda()] = -1
    pool.fork(other, lengths, torch.tensor([-1]).cuda())  # these entries' holder leaves
    assert int(pool.refs.sum()) == pages - len(gone)
    again = pool.reserve(other, lengths, len(gone) * 16)
    assert torch.equal(again[0, ::16].cpu() // 16, gone)


def test_tables_made_elsewhere(gpu):
    """hold counts a table's entries, shared ones and ones that are no page; rows of a wider table; entries never counted."""
    cache = KVCache.empty(50, 16, 2, 64, "int8")
    pool = PagePool(cache)
    wide = torch.tensor([[3, 7, -1, 9, 9], [3, 8, 50, 9, 9], [4, -7, 1 << 30, 9, 9]], dtype=torch.int32).cuda()
    table, lengths = wide[:, :3], _dev([20, 20, 5])
    pool.hold(table)
    want = [0] * 50
    for e in (3, 7, 3, 8, 4):
        want[e] += 1
    assert pool.refs.tolist() == want
    slots = pool.reserve(table, lengths, 13)  # row 2: its entry at column 1 is no page
    assert slots[0].tolist() == [7 * 16 + 4 + i for i in range(12)] + [0] and slots[2, :11].tolist() == [4 * 16 + 5 + i for i in range(11)]
    assert table[2].tolist()[:2] == [4, 2] and table[0].tolist() == [3, 7, 0] and table[1].tolist() == [3, 8, 1]
    assert (wide[:, 3:] == 9).all()
    fresh = torch.tensor([[6, -1]], dtype=torch.int32).cuda()  # an entry that nobody counted is no page of the row's
    assert pool.reserve(fresh, _dev([0]), 1).tolist() == [[5 * 16]] and fresh[0, 0] == 5


def test_part_of_a_table(gpu):
    """Rows forked and grown among themselves; their pages are shared with rows outside the call."""
    b = Both(60, 16, 6, 4)
    b.append(20)
    b.fork([0, 0, 0, 3, 4, 5])
    before = b.table.clone()
    part, ln = b.table[1:3], b.lengths[1:3]
    slots = b.pool.reserve(part, ln, 4)  # row 0 holds the pages too: both get copies
    assert torch.equal(b.table[0], before[0]) and torch.equal(b.table[3:], before[3:])
    assert len({int(t) for t in b.table[:3, 1]}) == 3 and (slots[:, 0] == b.table[1:3, 1].long() * 16 + 4).all()
    b.plain.table = b.table.tolist()
    assert b.pool.refs.tolist() == b.plain.refs()
    b.read()
    b.pool.fork(part, ln, torch.tensor([1, -1]).cuda())
    assert b.table[2].tolist() == [-1] * 4 and b.lengths[1:3].tolist() == [20, 0]
    b.plain.table = b.table.tolist()
    assert b.pool.refs.tolist() == b.plain.refs()


@pytest.mark.parametrize("S,width", [(1, 1), (1, 70), (255, 33), (257, 100), (1000, 17), (1024, 9), (1025, 9), (1300, 2100)])
def test_forks_of_every_size(gpu, S, width):
    """Few rows through LDS, many through a scratch table; against indexing."""
    g = torch.Generator().manual_seed(S + width)
    cache = KVCache.empty(500, 16, 1, 1, "bf16")
    pool = PagePool(cache)
    wide = torch.randint(-1, 500, (S, width + 3), generator=g).int().cuda()
    start, behind = wide[:, :width].clone(), wide[:, width:].clone()
    table, lengths = wide[:, :width], torch.randint(0, 999, (S,), generator=g).int().cuda()
    was = lengths.clone()
    pool.hold(table)
    parents = torch.randint(-1, S, (S,), generator=g).cuda()
    parents[::3] = torch.arange(S).cuda()[::3]
    parents[S // 2] = S
    pool.fork(table, lengths, parents)
    there = (parents >= 0) & (parents < S)
    want = torch.where(there[:, None], start[parents.clamp(0, S - 1)], -1)
    assert torch.equal(table, want) and torch.equal(wide[:, width:], behind)
    assert torch.equal(lengths, torch.where(there, was[parents.clamp(0, S - 1)], 0))
    assert torch.equal(pool.refs, torch.bincount(want[want >= 0].long(), minlength=500).int())
    free = torch.full((1, 500), -1, dtype=torch.int32).cuda()
    slots = pool.reserve(free, torch.zeros(1, dtype=torch.int32).cuda(), 500 * 16)[0, ::16] // 16
    n = int((torch.bincount(want[want >= 0].long(), minlength=500) == 0).sum())
    assert (slots >= 0).sum() == n and (pool.refs[slots[:n]] == 1).all()


def test_wide_tables(gpu):
    """Rows of more columns than a block takes."""
    width, S = 5000, 7
    cache = KVCache.empty(S * width + 9, 16, 1, 1, "bf16")
    pool = PagePool(cache)
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(S * width, generator=g).int().view(S, width).cuda()
    start, lengths = table.clone(), _dev([16 * width - 1] * S)
    pool.hold(table)
    parents = [3, 3, 0, 6, -1, 99, 6]
    pool.fork(table, lengths, _dev(parents, torch.int64))
    want = torch.stack([start[p] if 0 <= p < S else torch.full_like(start[0], -1) for p in parents])
    assert torch.equal(table, want)
    assert torch.equal(pool.refs, torch.bincount(want[want >= 0].long(), minlength=cache.pages).int())
    assert lengths.tolist() == [16 * width - 1 if 0 <= p < S else 0 for p in parents]
    slots = pool.reserve(table, lengths, 2)
    assert (slots[:, 1] == torch.tensor([-1, -1, -1, -1, -1, -1, -1]).cuda()).sum() == 5  # past the table


def _filled(pages, page, heads, dim, codes, seed, bounds):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = KVCache.empty(pages, page, heads, dim, codes)
    x = [torch.randn((pages * page, heads, dim), generator=g, device="cuda") for _ in range(2)]
    if cache.code >= 2:
        x = [t.to(cache.k.dtype) for t in x]
    cache.write(*x, torch.arange(pages * page, device="cuda"))
    b = PageBounds(cache, torch.randn((pages, heads, 2, cache.k.shape[3]), generator=g, device="cuda").bfloat16()) if bounds else None
    return cache, b


def _parts(cache, bounds):
    raw = [t.view(torch.uint8 if t.element_size() == 1 else torch.int16) for t in (cache.k, cache.v)]
    return raw + [t for t in (cache.k_scale, cache.v_scale) if t is not None] + ([] if bounds is None else [bounds.bounds])


@pytest.mark.parametrize("codes,heads,dim,page", [("int8", 3, 64, 16), ("fp8", 1, 200, 128), ("bf16", 2, 80, 32), ("fp16", 8, 256, 64)])
@pytest.mark.parametrize("with_bounds", [False, True])
def test_move(gpu, codes, heads, dim, page, with_bounds):
    for pages, room, live in ((70, 40, 31), (70, 20, 31), (5, 90, 5), (33, 33, 0), (1, 1, 1)):
        a, ab = _filled(pages, page, heads, dim, codes, 1, with_bounds)
        b, bb = _filled(room, page, heads, dim, codes, 2, with_bounds)
        g = torch.Generator().manual_seed(pages)
        used = torch.randperm(pages, generator=g)[:live]
        table = torch.full((3, max(live, 1) + 1), -1, dtype=torch.int32)
        table[0, :live] = used.int()
        table[1, :live // 2] = used[:live // 2].int()
        table = table.cuda()
        pool, into = PagePool(a, ab), PagePool(b, bb)
        into.hold(torch.arange(min(room, 3), dtype=torch.int32)[None].cuda())
        pool.hold(table)
        kept, refs, before = table.clone(), pool.refs.clone(), [t.clone() for t in _parts(a, ab)]
        old = [t.clone() for t in _parts(b, bb)]
        out = pool.move(table, into)
        order = used.sort().values
        to = {int(p): i for i, p in enumerate(order) if i < room}
        assert out.tolist() == [[to.get(e, -1) for e in r] for r in kept.tolist()]
        n = min(live, room)
        want = torch.zeros(room, dtype=torch.int32)
        want[:n] = refs.cpu()[order[:n]]
        assert torch.equal(into.refs.cpu(), want) and int(into.missing) == max(0, live - room)
        assert torch.equal(pool.refs, refs) and torch.equal(table, kept)
        for x, y, z, w in zip(_parts(a, ab), _parts(b, bb), before, old):
            assert torch.equal(x, z)
            assert torch.equal(y[:n], z[order[:n].cuda()]) and torch.equal(y[n:], w[n:])
        # its free pages are the ones behind
        more = torch.full((1, room + 1), -1, dtype=torch.int32).cuda()
        slots = into.reserve(more, _dev([0]), page * (room - n) + 1)
        assert (slots[0, ::page].cpu()[:room - n] // page == torch.arange(n, room)).all() and slots[0, -1] == -1


def test_move_of_many_pages(gpu):
    """More pages than a block's words of free bits cover."""
    pages = 32768 * 2 + 77
    a, b = KVCache.empty(pages, 16, 1, 1, "bf16"), KVCache.empty(pages - 5, 16, 1, 1, "bf16")
    a.k.view(pages, -1)[:, 0] = (torch.arange(pages) % 256).bfloat16().cuda()
    pool, into = PagePool(a), PagePool(b)
    g = torch.Generator().manual_seed(5)
    used = torch.randperm(pages, generator=g)[:pages // 2].sort().values.int()
    table = used[None].cuda()
    pool.hold(table)
    out = pool.move(table, into)
    assert torch.equal(out[0].cpu(), torch.arange(len(used), dtype=torch.int32))
    assert torch.equal(b.k.view(pages - 5, -1)[:len(used), 0], a.k.view(pages, -1)[table[0].long(), 0])
    assert (into.refs[:len(used)] == 1).all() and not into.refs[len(used):].any()
    assert into.reserve(torch.full((1, 2), -1, dtype=torch.int32).cuda(), _dev([0]), 1).tolist() == [[16 * len(used)]]


@pytest.mark.parametrize("codes,with_bounds", [("int8", True), ("bf16", False), ("fp16", True)])
def test_copy_pages(gpu, codes, with_bounds):
    a, ab = _filled(20, 32, 3, 100, codes, 3, with_bounds)
    b, bb = _filled(11, 32, 3, 100, codes, 4, with_bounds)
    want = [t.clone() for t in _parts(b, bb)]
    src, dst = [4, 19, 4, 20, 0, -1, 7], [0, 10, 5, 1, 11, 2, 3]
    for s, d in zip(src, dst):
        if 0 <= s < 20 and 0 <= d < 11:
            for x, y in zip(_parts(a, ab), want):
                y[d] = x[s]
    copy_pages(a, b, _dev(src, torch.int64), _dev(dst, torch.int64), ab, bb)
    assert all(torch.equal(x, y) for x, y in zip(_parts(b, bb), want))
    want = [t.clone() for t in _parts(a, ab)]
    for t in want:
        t[1], t[2] = t[8].clone(), t[8].clone()
    copy_pages(a, a, _dev([8, 8], torch.int64), _dev([1, 2], torch.int64), ab, ab)  # within one cache
    assert all(torch.equal(x, y) for x, y in zip(_parts(a, ab), want))
    none = torch.empty(0, dtype=torch.int64).cuda()
    copy_pages(a, b, none, none)


def test_pages_past_32_bits(gpu):
    """A cache of more than 2^32 bytes of keys: its last pages copied on a write, moved and copied."""
    page, heads, dim = 64, 8, 128
    pages = (1 << 32) // (page * heads * dim) + 40
    cache = KVCache.empty(pages, page, heads, dim, "int8")
    pool = PagePool(cache)
    far = pages - 1
    table = torch.tensor([[far, -1], [far, -1]], dtype=torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((10, heads, dim), generator=g, device="cuda")
    cache.write(x, -x, torch.arange(10, device="cuda") + far * page)
    pool.hold(table)
    most = torch.arange(pages - 2, dtype=torch.int32)[None].cuda()
    pool.hold(most)  # all but two pages are taken
    lengths = _dev([10, 10])
    slots = pool.reserve(table, lengths, 1)
    assert slots.tolist() == [[far * page + 10], [(pages - 2) * page + 10]]
    k, v = cache.read(cache.slots(table[1:], _dev([0]), 10)[0], torch.float32)
    assert torch.equal(k, cache.read(torch.arange(10, device="cuda") + far * page, torch.float32)[0]) and torch.equal(k, -v)
    small = KVCache.empty(3, page, heads, dim, "int8")
    copy_pages(cache, small, _dev([far], torch.int64), _dev([2], torch.int64))
    assert torch.equal(small.k[2], cache.k[far]) and torch.equal(small.v_scale[2], cache.v_scale[far])
    copy_pages(small, cache, _dev([2], torch.int64), _dev([pages - 3], torch.int64))
    assert torch.equal(cache.k[pages - 3], cache.k[far])


def test_captured_and_another_stream(gpu):
    """A beam step's fork and reservation in a graph: replayed, it goes on where the eager calls left the pool."""
    def make():
        b = Both(64, 16, 4, 6)
        b.append(21)
        return b

    one, two = make(), make()
    parents = torch.tensor([0, 0, 2, 1]).cuda()

    def step(b):
        b.pool.fork(b.table, b.lengths, parents)
        slots = b.pool.reserve(b.table, b.lengths, 1)
        b.lengths += 1
        return slots

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one)
    torch.cuda.current_stream().wait_stream(side)
    step(two)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(one)
    for i, p in enumerate(([0, 0, 2, 1], [3, 3, 3, 3], [1, 0, 3, 2], [2, -1, 2, 0], [0, 1, 1, 3])):
        parents.copy_(torch.tensor(p))
        want = step(two)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(one.table, two.table) and torch.equal(one.lengths, two.lengths)
        assert torch.equal(one.pool.refs, two.pool.refs) and torch.equal(one.cache.k, two.cache.k)


def test_nothing_to_do(gpu):
    cache = KVCache.empty(4, 16, 1, 64, "int8")
    pool = PagePool(cache)
    none = torch.empty((0, 3), dtype=torch.int32).cuda()
    pool.hold(none)
    pool.fork(none, _dev([]), _dev([], torch.int64))
    assert pool.reserve(none, _dev([]), 3).shape == (0, 3)
    table = torch.full((2, 3), -1, dtype=torch.int32).cuda()
    assert pool.reserve(table, _dev([0, 0]), 0).shape == (2, 0)
    assert pool.reserve(table, _dev([0, 0]), 4, _dev([0, -3])).tolist() == [[-1] * 4] * 2 and not pool.refs.any()
    assert pool.reserve(table, _dev([48, 1000]), 2).tolist() == [[-1] * 2] * 2 and not pool.refs.any()  # past the table
    assert int(pool.missing) == 0


def test_refusals(gpu):
    cache, other = KVCache.empty(4, 16, 2, 64, "int8"), KVCache.empty(4, 16, 2, 64, "fp8")
    pool = PagePool(cache)
    table, lengths, parents = torch.full((2, 3), -1, dtype=torch.int32).cuda(), _dev([0, 0]), torch.zeros(2, dtype=torch.int64).cuda()
    for bad in (table.long(), table.cpu(), table[0], table[:, :0], table.t(), table[:1].expand(2, 3)):
        with pytest.raises(ValueError):
            pool.hold(bad)
        with pytest.raises(ValueError):
            pool.reserve(bad, lengths, 1)
    for bad in (lengths.long(), lengths[:1], lengths.cpu(), _dev([0, 0, 0, 0])[::2]):
        with pytest.raises(ValueError):
            pool.fork(table, bad, parents)
        with pytest.raises(ValueError):
            pool.reserve(table, bad, 1)
    for bad in (parents.int(), parents[:1], parents.cpu()):
        with pytest.raises(ValueError):
            pool.fork(table, lengths, bad)
    for bad in (dict(count=-1), dict(count=1 << 30), dict(count=1, counts=lengths.long()), dict(count=1, counts=lengths[:1])):
        with pytest.raises(ValueError):
            pool.reserve(table, lengths, **bad)
    with pytest.raises(ValueError):
        pool.move(table, pool)
    with pytest.raises(ValueError):
        pool.move(table, PagePool(cache))
    with pytest.raises(ValueError):
        pool.move(table, PagePool(other))
    same = KVCache.empty(4, 16, 2, 64, "int8")
    with pytest.raises(ValueError):
        pool.move(table, PagePool(same, PageBounds(same)))
    with pytest.raises(ValueError):
        PagePool(cache, PageBounds(same))
    for a, b in ((parents, parents[:1]), (parents.int(), parents.int()), (parents.cpu(), parents.cpu()), (parents[None], parents[None])):
        with pytest.raises(ValueError):
            copy_pages(cache, same, a, b)
    with pytest.raises(ValueError):
        copy_pages(cache, other, parents, parents)
    with pytest.raises(ValueError):
        copy_pages(cache, same, parents, parents, PageBounds(cache))
    with pytest.raises(ValueError):
        copy_pages(cache, same, parents, parents, PageBounds(same), PageBounds(cache))
