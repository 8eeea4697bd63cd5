"""GPU: pages shared by rows of different lengths (ngram_amd.pages), after drafts that were not accepted or where pages ran out.
All comparisons are exact but for an 8-bit row's reading, which is one number and its scale's rounding."""

import pytest
import torch

from test_pages_gpu import Plain

from ngram_amd.kvcache import KVCache
from ngram_amd.pages import PagePool

pytestmark = pytest.mark.gpu


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


class Longest(Plain):
    """The pool's definition: where all that hold a page ask for it, the longest of them keeps it, of equal ones the first."""

    def reserve(self, count, counts=None):
        P, S = self.page, len(self.table)
        refs = self.refs()
        free = [g for g in range(self.pages) if refs[g] == 0]
        own = [count if counts is None else max(0, min(count, counts[r])) for r in range(S)]
        asks = [(r, c) for r in range(S) if own[r]
                for c in range(self.length[r] // P, min(self.width, (self.length[r] + own[r] - 1) // P + 1))]
        by = {}
        for r, c in asks:
            if self.table[r][c] >= 0:
                by.setdefault(self.table[r][c], []).append((r, c))
        keeps = {min(x, key=lambda a: (-self.length[a[0]], a)) for g, x in by.items() if len(x) == refs[g]}
        refused = set()
        for r, c in asks:
            if (r, c) in keeps:
                continue
            if not free:
                refused.add((r, c))
                continue
            self.table[r][c] = free.pop(0)
        self.missing += len(refused)
        return [[-1 if i >= own[r] or x // P >= self.width or (r, x // P) in refused else self.table[r][x // P] * P + x % P
                 for i, x in enumerate(range(n, n + count))] for r, n in enumerate(self.length)]


def _write(cache, numbers, slots):
    """Tokens that hold their numbers (below 251: exact in every type but for an 8-bit scale's rounding)."""
    x = numbers.reshape(-1, 1, 1).expand(-1, cache.heads, cache.dim).float() + 1
    x = x.to(cache.k.dtype if cache.code >= 2 else torch.float32).cuda()
    cache.write(x, -x, slots.reshape(-1))


def _read(cache, table, n):
    k, v = cache.read(cache.slots(table[None], _dev([0]), n)[0], torch.float32)
    return torch.stack([k, -v]) - 1


@pytest.mark.parametrize("codes", ["int8", "bf16"])
@pytest.mark.parametrize("others", [0, 600])  # the requests in a block's registers, and read again in each phase
def test_a_refused_row_keeps_its_tokens(gpu, codes, others):
    """Two rows of 5 and 10 tokens share the only page: the longer one goes on in it, behind the tokens of both."""
    cache = KVCache.empty(1, 16, 2, 5, codes)
    pool = PagePool(cache)
    S = 2 + others
    table = torch.full((S, 1), -1, dtype=torch.int32)
    table[:2] = 0
    table, lengths = table.cuda(), _dev([5, 10] + [0] * others)
    pool.hold(table)
    _write(cache, torch.arange(10), torch.arange(10).cuda())
    slots = pool.reserve(table, lengths, 1)
    assert slots[:2].tolist() == [[-1], [10]] and (slots[2:] == -1).all() and int(pool.missing) == 1 + others
    _write(cache, torch.arange(100, 100 + S), slots)
    want = torch.tensor([*range(10), 101]).cuda().view(1, -1, 1, 1)
    assert ((_read(cache, table[1], 11) - want).abs() < 0.5).all()
    assert ((_read(cache, table[0], 5) - want[:, :5]).abs() < 0.5).all()
    assert table[:2, 0].tolist() == [0, 0] and pool.refs.tolist() == [2]


@pytest.mark.parametrize("codes", ["int8", "fp8", "bf16"])
@pytest.mark.parametrize("page,rows,pages", [(16, 5, 14), (16, 12, 30), (32, 6, 9), (16, 90, 200), (16, 90, 900), (16, 700, 1500)])
def test_shared_pages_at_different_lengths(gpu, codes, page, rows, pages):
    """Forks, lengths cut back (drafts not accepted) and reservations in turn, with too few pages or enough: the pool is the
    definition's, and every row reads back its own past, refused ones too."""
    g = torch.Generator().manual_seed(rows + pages)
    width = 8
    cache = KVCache.empty(pages, page, 1, 5, codes)
    pool, plain = PagePool(cache), Longest(pages, page, rows, width)
    table, lengths = torch.full((rows, width), -1, dtype=torch.int32).cuda(), torch.zeros(rows, dtype=torch.int32).cuda()
    history, number = [[] for _ in range(rows)], 0
    for step in range(12):
        if step:
            parents = [int(x) if x < rows else -1 for x in torch.randint(0, rows + 2, (rows,), generator=g) // (1 + step % 3)]
            pool.fork(table, lengths, _dev(parents, torch.int64))
            plain.fork(parents)
            history = [list(history[p]) if p >= 0 else [] for p in parents]
            for s in range(rows):
                keep = max(0, len(history[s]) - int(torch.randint(0, page, (1,), generator=g)))
                del history[s][keep:]
                plain.length[s] = keep
            lengths.copy_(_dev(plain.length))
        count = int(torch.randint(1, page + 3, (1,), generator=g))
        counts = torch.randint(-1, count + 1, (rows,), generator=g).tolist() if step % 2 else None
        slots = pool.reserve(table, lengths, count, None if counts is None else _dev(counts))
        want = plain.reserve(count, counts)
        assert slots.tolist() == want and table.tolist() == plain.table
        assert pool.refs.tolist() == plain.refs() and int(pool.missing) == plain.missing
        numbers = torch.arange(number, number + rows * count).view(rows, count) % 251
        number += rows * count
        _write(cache, numbers, slots)
        for s in range(rows):
            n = next((i for i, x in enumerate(want[s]) if x < 0), count)
            history[s] += numbers[s, :n].tolist()
            plain.length[s] += n
        lengths.copy_(_dev(plain.length))
        for s in range(rows):
            if history[s]:
                got = _read(cache, table[s], len(history[s]))
                assert ((got - torch.tensor(history[s]).cuda().view(1, -1, 1, 1)).abs() < 0.5).all(), (step, s)
