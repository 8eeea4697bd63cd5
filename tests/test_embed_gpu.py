"""GPU: embedded hint rows (ngram_amd.embed) against the definition in float64, with the table's and the weights'
gradients: element types, row lengths that are odd or not whole loads, slots, entries that do not count (weight 0, no
cell) over table rows that hold NaN, tokens outside the table, tokens so frequent that their gradient is summed in pieces,
strided tables and gradients, empty batches, streams, and the refusals.

Tolerances (u the unit roundoff of the element type, 2^-24 that of the 32-bit sums): a sum of c products held in 32 bits is
off by at most (c + 2) 2^-24 times the sum of the terms' sizes, and rounding it once by u of itself (or half the smallest
subnormal)."""

import numpy as np
import pytest
import torch

from ngram_amd import hints as H
from ngram_amd.embed import HintEmbedding, embed

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}


def _case(seed, V, n, slots, entries, dim, dtype, skew=1.0, token_type=torch.int64, cell_type=torch.int64):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn((V, dim), generator=g).to(dtype)
    lead = (n,) if slots == 1 else (n, slots)
    tokens = (torch.rand((*lead, entries), generator=g) ** skew * V).long().clamp(max=V - 1)
    weights = torch.rand((*lead, entries), generator=g) * (torch.rand((*lead, entries), generator=g) < 0.6)
    cell = torch.randint(0, 3, lead, generator=g)
    up = torch.randn((n, dim), generator=g).to(dtype)
    return table, tokens.to(token_type), weights, cell.to(cell_type), up


def _definition(table, tokens, weights, cell, up, scale):
    """out, grad, slopes in float64 with the sums of their terms' sizes and counts."""
    V, dim = table.shape
    n = tokens.shape[0]
    t = table.double().nan_to_num(0.0)
    tok = tokens.long().reshape(n, -1)
    w = weights.double().reshape(n, -1)
    has = (cell > 0).reshape(n, -1).repeat_interleave(tokens.shape[-1], 1)
    counted = has & (w != 0)
    w = torch.where(counted, w, 0.0)
    rows = t[tok]
    out, size = (w[..., None] * rows).sum(1) * scale, (w[..., None] * rows).abs().sum(1) * scale
    u = up.double()
    grad, gsize = torch.zeros((V, dim)).double(), torch.zeros((V, dim)).double()
    terms = (w[..., None] * u[:, None]).reshape(-1, dim)
    grad.index_add_(0, tok.reshape(-1), terms)
    gsize.index_add_(0, tok.reshape(-1), terms.abs())
    many = torch.zeros(V).double().index_add_(0, tok.reshape(-1), counted.reshape(-1).double())
    slopes = (rows * u[:, None]).sum(-1) * has * scale
    ssize = (rows * u[:, None]).abs().sum(-1) * has * scale
    return (out, size, tok.shape[1]), (grad * scale, gsize * scale, many[:, None]), (slopes, ssize, dim)


def _check(got, want, size, count, dtype, what):
    got = got.double().cpu()
    bound = U[dtype] * want.abs() + (count + 4) * 2.0**-24 * size * (1 + U[dtype]) + TINY[dtype]
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound).all(), (what, float((off - bound).max()), float(off.max()))


def _run(table, tokens, weights, cell, up, scale, learned=True):
    t = table.cuda().requires_grad_(True)
    w = weights.cuda().requires_grad_(learned)
    out = embed(t, tokens.cuda(), w, None if cell is None else cell.cuda(), scale)
    grads = torch.autograd.grad(out, [t, w] if learned else [t], up.cuda())
    return out.detach(), *grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,slots,entries,dim", [(1, 1, 1, 1), (3, 1, 8, 64), (130, 2, 8, 333), (257, 1, 5, 768),
                                                 (64, 3, 30, 40), (33, 1, 8, 1030), (1000, 1, 8, 100)])
def test_rows_and_gradients(gpu, dtype, n, slots, entries, dim):
    args = _case(n + dim, 301, n, slots, entries, dim, dtype)
    out, grad, slopes = _run(*args, 0.75)
    (o, g, s) = _definition(*args, 0.75)
    assert out.dtype == dtype and grad.dtype == dtype and grad.shape == args[0].shape and slopes.shape == args[2].shape
    _check(out, *o, dtype, "out")
    _check(grad, *g, dtype, "grad")
    _check(slopes.reshape(n, -1), *s, torch.float32, "slopes")


@pytest.mark.parametrize("token_type", [torch.int32, torch.uint16])
@pytest.mark.parametrize("cell_type", [torch.int32, torch.int16])
def test_types_of_tokens_and_cells(gpu, token_type, cell_type):
    args = _case(5, 60000, 200, 2, 8, 96, torch.bfloat16, token_type=token_type, cell_type=cell_type)
    out, grad, _ = _run(*args, 1.0)
    o, g, _ = _definition(*args, 1.0)
    _check(out, *o, torch.bfloat16, "out")
    _check(grad, *g, torch.bfloat16, "grad")


@pytest.mark.parametrize("V,skew", [(1, 1.0), (3, 1.0), (500, 6.0), (70000, 30.0)])
@pytest.mark.parametrize("dtype,dim", [(torch.float32, 65), (torch.bfloat16, 256)])
def test_frequent_tokens(gpu, V, skew, dtype, dim):
    """Tokens with hundreds of entries beside absent ones: runs over many chunks of the sorted list, starting and ending
    anywhere in one."""
    args = _case(V, V, 1501, 1, 8, dim, dtype, skew=skew)
    out, grad, slopes = _run(*args, 1.5)
    o, g, s = _definition(*args, 1.5)
    _check(grad, *g, dtype, "grad")
    _check(out, *o, dtype, "out")
    again = _run(*args, 1.5)
    assert torch.equal(grad, again[1]) and torch.equal(slopes, again[2])  # the same on every run


@pytest.mark.parametrize("run", [63, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("before", [0, 1, 63, 64, 65])
def test_runs_at_chunk_ends(gpu, run, before):
    """One token's run of entries at every place of the sorted list's chunks."""
    tokens = torch.cat([torch.zeros(before), torch.full((run,), 1), torch.full((70,), 2)]).long()
    tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(run))]
    up = torch.randn((len(tokens), 32), generator=torch.Generator().manual_seed(before))
    t = torch.randn(4, 32).cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(embed(t, tokens.cuda()), [t], up.cuda())
    want = torch.zeros(4, 32).double().index_add_(0, tokens, up.double())
    size = torch.zeros(4, 32).double().index_add_(0, tokens, up.double().abs())
    _check(grad, want, size, 200, torch.float32, "grad")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,dim", [((1,), 1), ((7,), 768), ((3, 50), 33), ((1025,), 64), ((0,), 16)])
def test_lookup(gpu, dtype, shape, dim):
    g = torch.Generator().manual_seed(dim)
    table = torch.randn((97, dim), generator=g).to(dtype)
    tokens = torch.randint(0, 97, shape, generator=g)
    up = torch.randn((*shape, dim), generator=g).to(dtype)
    t = table.cuda().requires_grad_(True)
    out = embed(t, tokens.cuda(), scale=3.0)
    assert torch.equal(out.detach().cpu(), (table.float() * 3.0).to(dtype)[tokens])  # one product, rounded once
    (grad,) = torch.autograd.grad(out, [t], up.cuda())
    flat, u = tokens.reshape(-1), up.double().reshape(-1, dim)
    want = torch.zeros(97, dim).double().index_add_(0, flat, u) * 3
    size = torch.zeros(97, dim).double().index_add_(0, flat, u.abs()) * 3
    _check(grad, want, size, int(np.prod(shape)), dtype, "grad")


def test_entries_that_do_not_count_are_not_read(gpu):
    """Table rows of NaN and tokens outside the table behind weight 0 or a slot without a cell: nothing of them shows."""
    table, tokens, weights, cell, up = _case(1, 50, 400, 2, 8, 72, torch.float32)
    dead = (weights == 0) | (cell <= 0)[..., None]
    table[7] = float("nan")
    tokens = torch.where(dead, torch.where(tokens % 2 == 0, 7, 1 << 40), torch.where(tokens == 7, 8, tokens))
    clean = torch.where(dead, 0, tokens)
    out, grad, _ = _run(table, tokens, weights, cell, up, 1.0, learned=True)
    o, g, _ = _definition(table, clean, weights, cell, up, 1.0)
    _check(out, *o, torch.float32, "out")
    _check(grad, *g, torch.float32, "grad")


def test_negative_weights_and_cells(gpu):
    table, tokens, weights, cell, up = _case(2, 50, 300, 1, 8, 72, torch.float32)
    weights, cell = weights - 0.3, cell - 1
    out, grad, slopes = _run(table, tokens, weights, cell, up, -2.0)
    o, g, s = _definition(table, tokens, weights, cell, up, -2.0)
    for got, (want, size, count), what in ((out, o, "out"), (grad, g, "grad"), (slopes.reshape(300, -1), s, "slopes")):
        _check(got, want, size.abs(), count, torch.float32, what)


@pytest.mark.parametrize("bad", [-1, 50, 1 << 35])
def test_a_counted_token_outside_the_table(gpu, bad):
    table, tokens, weights, cell, up = _case(3, 50, 40, 1, 8, 72, torch.float32)
    cell[:] = 1
    tokens[11, 3], weights[11, 3] = bad, 0.5
    out, grad, slopes = _run(table, tokens, weights, cell, up, 1.0)
    assert torch.isnan(out[11]).all() and torch.isfinite(out[torch.arange(40) != 11]).all()
    assert torch.isfinite(grad).all() and int(torch.isnan(slopes).sum()) == 1 and torch.isnan(slopes[11, 3])
    clean = tokens.clone()
    clean[11, 3], weights[11, 3] = 0, 0.0
    _, g, _ = _definition(table, clean, weights, cell, up, 1.0)
    _check(grad, *g, torch.float32, "grad")
    t = table.cuda().requires_grad_(True)
    look = embed(t, tokens.cuda()[:, 3])
    assert torch.isnan(look[11]).all() and torch.isfinite(look[:11]).all()


def test_strides(gpu):
    """A table with a row stride, at an odd offset; gradients that are expanded, transposed or strided."""
    table, tokens, weights, cell, up = _case(4, 60, 100, 1, 8, 48, torch.bfloat16)
    wide = torch.zeros((60, 101), dtype=torch.bfloat16)
    wide[:, 3:51] = table
    t = wide.cuda()[:, 3:51].requires_grad_(True)
    out = embed(t, tokens.cuda(), weights.cuda(), cell.cuda())
    o, g, _ = _definition(table, tokens, weights, cell, up, 1.0)
    _check(out.detach(), *o, torch.bfloat16, "out")
    for u in (up.cuda().t().contiguous().t(), torch.cat([up, up], 1).cuda()[:, :48]):
        (grad,) = torch.autograd.grad(out, [t], u, retain_graph=True)
        _check(grad, *g, torch.bfloat16, "grad")
    (grad,) = torch.autograd.grad(out.float().sum(), [t])  # an expanded gradient
    _, g, _ = _definition(table, tokens, weights, cell, torch.ones_like(up), 1.0)
    _check(grad, *g, torch.bfloat16, "grad of the sum")
    by_column = tokens.cuda().t().contiguous().t()  # tokens in another memory order
    assert torch.equal(embed(t, by_column, weights.cuda(), cell.cuda()), out)


def test_gradients_against_differences(gpu):
    """d<out, up> along a random direction of table and weights against central differences of the operator itself in
    float32: out is linear in each, so a difference over 2 h is exact up to rounding, 2^-24 (4 terms) over h a term."""
    table, tokens, weights, cell, up = _case(6, 40, 60, 2, 8, 33, torch.float32)
    t, w = table.cuda().requires_grad_(True), weights.cuda().requires_grad_(True)
    tok, c, u = tokens.cuda(), cell.cuda(), up.cuda()
    dt, dw = torch.autograd.grad(embed(t, tok, w, c, 0.5), [t, w], u)
    g = torch.Generator().manual_seed(9)
    a = torch.randn(table.shape, generator=g).cuda()
    b = (torch.randn(weights.shape, generator=g) * (weights != 0)).cuda()  # entries of weight 0 stay uncounted

    def at(x, y):
        return (embed(t.detach() + x, tok, w.detach() + y, c, 0.5).double() * u.double()).sum()

    zero_t, zero_w, h = torch.zeros_like(a), torch.zeros_like(b), 0.25
    size = float((embed(t.detach().abs() + a.abs(), tok, w.detach() + b.abs(), c, 0.5).double() * u.abs().double()).sum())
    bound = size * 2.0**-24 * 4 * (16 + 4) / h
    assert abs(float((at(h * a, zero_w) - at(-h * a, zero_w)) / (2 * h) - (dt.double() * a.double()).sum())) < bound
    assert abs(float((at(zero_t, h * b) - at(zero_t, -h * b)) / (2 * h) - (dw.double() * b.double()).sum())) < bound


def test_large_rows_of_entries(gpu):
    """More entries a position than a wave has lanes."""
    args = _case(8, 90, 50, 3, 70, 65, torch.float32)
    out, grad, slopes = _run(*args, 1.0)
    o, g, s = _definition(*args, 1.0)
    _check(out, *o, torch.float32, "out")
    _check(grad, *g, torch.float32, "grad")
    _check(slopes.reshape(50, -1), *s, torch.float32, "slopes")


def test_empty_batch_and_empty_rows(gpu):
    t = torch.randn(9, 16).cuda().requires_grad_(True)
    none = torch.zeros((0, 8), dtype=torch.int64).cuda()
    out = embed(t, none, torch.zeros((0, 8)).cuda(), none[:, 0])
    assert out.shape == (0, 16)
    (grad,) = torch.autograd.grad(out.sum(), [t])
    assert torch.equal(grad, torch.zeros_like(t))
    tok = torch.zeros((5, 8), dtype=torch.int64).cuda()
    for w, c in ((torch.zeros(5, 8), torch.ones(5)), (torch.ones(5, 8), torch.zeros(5))):
        out = embed(t, tok, w.cuda(), c.long().cuda())
        (grad,) = torch.autograd.grad(out.sum(), [t])
        assert not out.any() and not grad.any()


def test_another_stream_and_a_module(gpu):
    """HintEmbedding over fake hint rows, its step run on a stream of its own."""
    import os

    os.environ.pop("HINT_NGRAM", None)
    rows = H.Hints("fake").val_span(0, 3000)
    torch.manual_seed(1)
    e = HintEmbedding(H.VOCAB, 96, scale=0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = e(rows)
        out.square().sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    up = 2 * out.detach()
    o, g, _ = _definition(e.weight.detach().cpu(), rows.tokens.cpu(), rows.weights.cpu(), rows.cell.cpu(), up.cpu(), 0.5)
    _check(out.detach(), *o, torch.float32, "out")
    _check(e.weight.grad, *g, torch.float32, "grad")


def test_refusals(gpu):
    t = torch.randn(9, 16).cuda()
    tok = torch.zeros((5, 8), dtype=torch.int64).cuda()
    w, c = torch.ones(5, 8).cuda(), torch.ones(5, dtype=torch.int64).cuda()
    bad = [
        (t.double(), tok, w, c), (t[0], tok, w, c), (t.t(), tok, w, c), (t.cpu(), tok, w, c), (t, tok.cpu(), w, c),
        (t, tok.float(), w, c), (t, tok, w.double(), c), (t, tok, w[:, :7], c), (t, tok, w, c[:4]), (t, tok, w, c.float()),
        (t, tok, None, c), (t, tok[0], w[0], None), (t, tok[:, :0], w[:, :0], c), (t[:0], tok, w, c),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            embed(*args)
    with pytest.raises(ValueError):
        embed(t, tok, w, c, float("nan"))
    with pytest.raises(ValueError):
        embed(t, tok[:1, :1].expand(1 << 20, 1 << 11), w[:1, :1].expand(1 << 20, 1 << 11))


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 72), (torch.bfloat16, 300)])
def test_weights_gradient_of_entries_that_do_not_count(gpu, dtype, dim):
    """Padding: a weight of 0, or a slot without a cell, before a token outside the table. Its slope is 0 as everything of
    it; a weight of 0 before a token of the table has the slope that it would count with; without a cell, 0."""
    table, tokens, weights, cell, up = _case(21, 50, 400, 2, 8, dim, dtype)
    dead = (weights == 0) | (cell <= 0)[..., None]
    outside = dead & (torch.rand(dead.shape, generator=torch.Generator().manual_seed(1)) < 0.5)
    assert (outside & (weights == 0) & (cell > 0)[..., None]).any() and (dead & ~outside).any()
    far = torch.tensor([-1, 50, 1 << 40])[torch.arange(outside.numel()).reshape(outside.shape) % 3]
    out, grad, slopes = _run(table, torch.where(outside, far, tokens), weights, cell, up, 0.5)
    o, g, (want, size, count) = _definition(table, tokens, weights, cell, up, 0.5)
    _check(out, *o, dtype, "out")
    _check(grad, *g, dtype, "grad")
    off = outside.reshape(want.shape)
    assert not slopes.cpu().reshape(want.shape)[off].any()  # 0, not NaN
    _check(torch.where(off.cuda(), 0.0, slopes.reshape(want.shape)), torch.where(off, 0.0, want),
           torch.where(off, 0.0, size), count, torch.float32, "slopes")


def test_forward_mode_is_refused(gpu):
    """There is no forward-mode derivative: a tangent raises instead of being lost."""
    import torch.autograd.forward_ad as fw

    table, tokens, weights, cell, up = (x.cuda() for x in _case(23, 50, 40, 1, 8, 72, torch.float32))
    want = embed(table, tokens, weights, cell)
    with fw.dual_level():
        for t, w in ((fw.make_dual(table, table), weights), (table, fw.make_dual(weights, weights))):
            with pytest.raises(RuntimeError, match="jvp"):
                embed(t, tokens, w, cell)
        with pytest.raises(RuntimeError, match="jvp"):
            embed(fw.make_dual(table, table), tokens)
        assert torch.equal(embed(table, tokens, weights, cell), want)


def test_scales_that_are_no_float32_are_refused(gpu):
    t, tok = torch.randn(9, 16).cuda(), torch.zeros(5, dtype=torch.int64).cuda()
    for scale in (1e39, -1e39, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            embed(t, tok, scale=scale)


def _sums(V, tok, up):
    want = torch.zeros((V, up.shape[1]), device="cuda", dtype=torch.float64).index_add_(0, tok, up.double())
    size = torch.zeros_like(want).index_add_(0, tok, up.double().abs())
    return want, size, torch.zeros((V, 1), device="cuda", dtype=torch.float64).index_add_(
        0, tok, torch.ones((len(tok), 1), device="cuda", dtype=torch.float64))


def _check_sums(grad, tok, up):
    want, size, many = _sums(grad.shape[0], tok, up)
    bound = 2.0**-24 * want.abs() + (many + 4) * 2.0**-24 * size * (1 + 2.0**-24) + 2.0**-149
    assert ((grad.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [(1 << 21) + 1, 3000001])
def test_gradient_of_many_entries(gpu, n):
    """More than 2^21 entries: the sort's spans grow past their smallest."""
    g = torch.Generator(device="cuda").manual_seed(n)
    V = 70001
    tok = (torch.rand(n, generator=g, device="cuda") ** 3 * V).long().clamp_(max=V - 1)
    up = torch.randn((n, 4), generator=g, device="cuda")
    t = torch.zeros((V, 4), device="cuda", requires_grad=True)
    (grad,) = torch.autograd.grad(embed(t, tok), [t], up)
    _check_sums(grad, tok, up)


@pytest.mark.parametrize("n", [300, 50001])
def test_gradient_of_a_table_past_24_bits(gpu, n):
    """More than 2^24 rows: a fourth pass of digits, by one block and by many."""
    g = torch.Generator(device="cuda").manual_seed(n)
    V = (1 << 24) + 1001
    tok = torch.randint(0, V, (n,), generator=g, device="cuda")
    tok[:200] = V - 1 - tok[:200] % 7
    tok[200:220] = tok[200:220] % 1000 + (1 << 24)
    up = torch.randn((n, 2), generator=g, device="cuda")
    t = torch.zeros((V, 2), device="cuda", requires_grad=True)
    (grad,) = torch.autograd.grad(embed(t, tok), [t], up)
    _check_sums(grad, tok, up)
