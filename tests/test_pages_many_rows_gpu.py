"""GPU: forks of very many rows (ngram_amd.pages): against indexing, and how their time grows."""

import pytest
import torch

from ngram_amd.kvcache import KVCache
from ngram_amd.pages import PagePool

pytestmark = pytest.mark.gpu


def _fork_ms(S):
    cache = KVCache.empty(64, 16, 1, 1, "bf16")
    pool = PagePool(cache)
    table = torch.randint(0, 64, (S, 2), generator=torch.Generator().manual_seed(S)).int().cuda()
    lengths = torch.arange(S, dtype=torch.int32).cuda()
    parents = torch.randint(-1, S + 1, (S,), generator=torch.Generator().manual_seed(1)).cuda()
    pool.hold(table)
    start, times = table.clone(), []
    for i in range(4):
        table.copy_(start)
        lengths.copy_(torch.arange(S))
        pool.clear()
        pool.hold(table)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        pool.fork(table, lengths, parents)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    there = (parents >= 0) & (parents < S)
    want = torch.where(there[:, None], start[parents.clamp(0, S - 1)], -1)
    assert torch.equal(table, want) and torch.equal(lengths.long(), torch.where(there, parents, 0))
    assert torch.equal(pool.refs, torch.bincount(want[want >= 0].long(), minlength=64).int())
    return min(times)


@pytest.mark.parametrize("S", [1025, 4095, 4096, 4097, 70001])
def test_forks_of_many_rows(gpu, S):
    _fork_ms(S)


def test_forks_of_very_many_rows(gpu):
    """A fork's time grows with its rows, not with their square (16 times for four times the rows)."""
    few, many = _fork_ms(1 << 16), _fork_ms(1 << 18)
    assert many < 8 * few, (few, many)
