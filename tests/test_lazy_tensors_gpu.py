"""GPU: tensors that torch conjugates or negates by a bit, their memory left as it is, as inputs of the model's and the decoding
operators."""

import pytest
import torch

from ngram_amd.beam import beam_step, reorder
from ngram_amd.kvcache import KVCache
from ngram_amd.sparse import PageBounds, sparse_attention
from ngram_amd.tree import tree_attention

pytestmark = pytest.mark.gpu


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128, torch.complex32])
def test_reorder_of_lazy_states(gpu, dtype):
    """torch conjugates and negates by a bit of the tensor: the states' values are those that torch shows."""
    g = torch.Generator(device="cuda").manual_seed(2)
    real = {torch.complex32: torch.float16, torch.complex64: torch.float32, torch.complex128: torch.float64}[dtype]
    z = torch.view_as_complex(torch.randn((6, 7, 2), generator=g, device="cuda").to(real))
    assert z.dtype == dtype
    parents = _dev([3, 3, 0, 5, -1], torch.int64)

    def same(state):
        got, want = reorder(state, parents), state.resolve_conj().resolve_neg()[parents.clamp(min=0)]
        want[-1] = 0
        assert got.dtype == state.dtype and not got.is_conj() and not got.is_neg()
        assert torch.equal(got, want) if not got.is_complex() else torch.equal(torch.view_as_real(got), torch.view_as_real(want))

    for state in (z, z.conj(), z.conj()[:, 2:5], z.conj().imag, z.conj()[:, 3].imag, z.conj().imag[:, 3], z.t().contiguous().t().conj()):
        same(state)
    assert all(torch.equal(a.real, b) for a, b in zip(reorder([z.conj(), z], parents), [reorder(z, parents).real] * 2))


def test_lazily_negated_inputs(gpu):
    """Rows of one element, which are contiguous whatever their stride."""
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.view_as_complex(torch.randn((2, 3, 4, 1, 2), generator=g, device="cuda").half())
    q = z.conj().imag  # [2, 3, 4, 1], negated by a bit
    assert q.is_neg()
    cache = KVCache.empty(8, 16, 2, 1, "fp16")
    x = torch.randn((8 * 16, 2, 1), generator=g, device="cuda").half()
    cache.write(x, x, torch.arange(8 * 16, device="cuda"))
    bounds = PageBounds(cache)
    table, lengths = torch.arange(8, dtype=torch.int32).view(2, 4).cuda(), _dev([50, 61])
    bounds.update(table, _dev([0, 0]), 64)
    a, b = (sparse_attention(t, cache, bounds, table, lengths, 2, return_pages=True) for t in (q, q.resolve_neg()))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(tree_attention(q, cache, table, lengths), tree_attention(q.resolve_neg(), cache, table, lengths))
    for n in (1, 5):
        k = torch.view_as_complex(torch.randn((n, 1, 1, 2), generator=g, device="cuda")).conj().imag
        one = KVCache.empty(1, 16, 1, 1, "int8")
        one.write(k, k, torch.arange(n, device="cuda"))
        assert k.is_neg() and all((t[:, 0, 0] - k[:, 0, 0]).abs().max() < 1e-5 for t in one.read(torch.arange(n, device="cuda"), torch.float32))
    logits, scores = z.conj().imag[..., 0], torch.zeros((2, 3)).cuda()
    for t in (logits, logits[..., :1]):
        a, b = (beam_step(s, scores) for s in (t, t.resolve_neg()))
        assert torch.equal(a.scores, b.scores) and torch.equal(a.tokens, b.tokens)
