"""GPU: a beam search's step (ngram_amd.beam) against its definition in float64: element types, sizes around the chunks' and
blocks', ties, masked tokens, finished beams, lengths, too few candidates, NaN and infinities, strides, streams, graphs, and the
refusals; the states' reordering.

Tolerances. A row's log-sum: a term 2^t beside the largest (1) has its exponent rounded once, off by |t| 2^-24, so itself by
0.7 |t| 2^-24, and the instruction adds 2^-23; of V <= 2^17 terms those with |t| > 20 weigh less than 2^-3 of the largest
together and less the further they lie, so a sum is off by 20 * 0.7 * 2^-24 < 2^-20 and 2^-23 of itself at most; a thread's
sum of up to 32 terms adds 31 * 2^-24, the rest is 64 bits: LSE = 2^-20 + 2^-23 + 31 * 2^-24. A score is rounded to float32
once: 2^-24 of itself more. Two candidates may come in the other order where their exact ranks differ by less than twice LSE
(over their lengths' norms, which are 1 at least); within a beam the order is the logits'."""

import math

import pytest
import torch

from ngram_amd.beam import beam_step, reorder

pytestmark = pytest.mark.gpu

LSE = 2.0**-20 + 2.0**-23 + 31 * 2.0**-24


def _ranked(logits, scores, lengths, finished, pad, alpha):
    """Per sequence: its candidates as (rank, beam, logit, token, total), best first."""
    B, W, V = logits.shape
    lp = logits.double().cpu()
    lse = torch.logsumexp(lp, 2)
    out = []
    for b in range(B):
        rows = []
        for w in range(W):
            s = float(scores[b, w])
            done = finished is not None and bool(finished[b, w])
            n = 0 if lengths is None else int(lengths[b, w])
            norm = max(n + (0 if done else 1), 1) ** alpha
            if done:
                totals = [(math.inf, pad, s)]
            else:
                x, z = lp[b, w].tolist(), float(lse[b, w])
                if math.isnan(z) or math.isinf(z):
                    continue
                totals = [(l, v, s + (l - z)) for v, l in enumerate(x)]
            rows += [(t / norm, w, l, v, t) for l, v, t in totals if t / norm > -math.inf]
        rows.sort(key=lambda r: (-r[0], r[1], -r[2], r[3]))
        out.append(rows)
    return out


def _check(step, logits, scores, lengths=None, finished=None, keep=None, end=None, pad=None, alpha=0.0):
    B, W, V = logits.shape
    K = W if keep is None else keep
    pad = end if pad is None else pad
    assert step.scores.shape == step.parents.shape == step.tokens.shape == (B, K)
    ranked = _ranked(logits, scores, lengths, finished, pad, alpha)
    got = [t.tolist() if t is not None else None for t in step]
    for b in range(B):
        rows, seen = ranked[b], {}
        by = {(r[1], r[3]): r for r in rows}
        spare = (i for i in range(W * V) if (i // V, i % V) not in by)
        last = {}
        for k in range(K):
            w, v = got[1][b][k] - b * W, got[2][b][k]
            assert 0 <= w < W and 0 <= v < V and (w, v) not in seen
            seen[w, v] = True
            done = finished is not None and bool(finished[b, w])
            if got[3] is not None:
                assert got[3][b][k] == (done or v == end)
            if got[4] is not None:
                assert got[4][b][k] == int(lengths[b, w]) + (0 if done else 1)
            if k >= len(rows):
                i = next(spare)
                assert (w, v) == (i // V, i % V) and got[0][b][k] == -math.inf
                continue
            r, want = by[w, v], rows[k]
            assert (r[1], r[3]) == (want[1], want[3]) or abs(r[0] - want[0]) <= 2 * LSE, (b, k, r, want)
            if math.isinf(r[4]):
                assert got[0][b][k] == r[4]
            else:
                assert abs(got[0][b][k] - r[4]) <= LSE + 2.0**-24 * abs(r[4])
            if w in last:  # the order within a beam is exact
                assert (-last[w][0], last[w][1]) < (-r[2], r[3])
            last[w] = r[2], r[3]


def _inputs(seed, B, W, V, dtype, ended=0.0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((B, W, V), generator=g) * spread).to(dtype).cuda()
    scores = (-torch.rand((B, W), generator=g) * 6 - 1).cuda()
    lengths = torch.randint(0, 30, (B, W), generator=g, dtype=torch.int32).cuda()
    finished = (torch.rand((B, W), generator=g) < ended).cuda()
    return logits, scores, lengths, finished


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,W,V,K", [(1, 1, 1, 1), (1, 4, 50257, 4), (3, 2, 257, 5), (2, 5, 2047, 5), (2, 3, 2049, 6), (1, 8, 8193, 16),
                                     (7, 1, 1000, 1), (2, 128, 300, 128), (1, 32, 20011, 64), (2, 9, 16, 128), (1, 2, 100003, 3)])
def test_shapes(gpu, dtype, B, W, V, K):
    logits, scores, lengths, finished = _inputs(V + K, B, W, V, dtype, 0.2)
    step = beam_step(logits, scores, lengths, finished, keep=K, end=V - 1, alpha=0.6)
    _check(step, logits, scores, lengths, finished, K, V - 1, None, 0.6)
    step = beam_step(logits, scores, keep=K)  # no ends, no lengths
    assert step.finished is None and step.lengths is None
    _check(step, logits, scores, None, None, K)


@pytest.mark.parametrize("B,W,V", [(130, 8, 8192), (40, 8, 33000)])  # chunks of 8192 and of fewer
def test_many_rows(gpu, B, W, V):
    logits, scores, lengths, finished = _inputs(B, B, W, V, torch.bfloat16, 0.3)
    step = beam_step(logits, scores, lengths.long(), finished, end=0, pad=7, alpha=1.0)
    assert step.lengths.dtype == torch.int64
    few = slice(B - 3, B)  # the definition of every row takes long
    part = type(step)(*(t[few] for t in step))
    part = part._replace(parents=part.parents - (B - 3) * W)
    _check(part, logits[few], scores[few], lengths[few], finished[few], None, 0, 7, 1.0)
    assert ((step.parents // W).cpu() == torch.arange(B)[:, None]).all()


@pytest.mark.parametrize("V,K", [(50257, 8), (8192, 128), (300, 128), (70000, 100)])
def test_ties_go_to_the_lower_token(gpu, V, K):
    """All logits alike; a few distinct values; many beams alike."""
    same = torch.zeros((1, 1, V), dtype=torch.bfloat16).cuda()
    scores = torch.zeros((1, 1)).cuda()
    step = beam_step(same, scores, keep=K)
    assert torch.equal(step.tokens[0].cpu(), torch.arange(K))
    g = torch.Generator().manual_seed(K)
    few = torch.randint(-2, 3, (1, 1, V), generator=g).half().cuda()
    step = beam_step(few, scores, keep=K)
    want = torch.sort(few[0, 0].float().cpu(), descending=True, stable=True).indices[:K]
    assert torch.equal(step.tokens[0].cpu(), want)
    zeros = torch.zeros(V)  # 0 and -0 are alike
    zeros[::2] = -0.0
    assert torch.equal(beam_step(zeros.view(1, 1, V).cuda(), scores, keep=K).tokens[0].cpu(), torch.arange(K))
    alike = few.expand(1, 6, V)
    step = beam_step(alike, torch.zeros((1, 6)).cuda(), keep=K)  # equal ranks: the lower beam, then the lower token
    top = (few[0, 0] == few.max()).nonzero()[:, 0].cpu()
    order = [(w, int(v)) for w in range(6) for v in top[:K]][:K]
    assert [(int(p), int(t)) for p, t in zip(step.parents[0], step.tokens[0])] == order[:K] or len(top) * 6 < K


def test_masked_tokens_and_beams(gpu):
    """Allowed tokens only (the others -inf), dead beams, a search's start; too few candidates."""
    logits, scores, lengths, _ = _inputs(5, 3, 4, 9001, torch.float32)
    allowed = [3, 77, 8999, 9000]
    masked = torch.full_like(logits, -math.inf)
    masked[..., allowed] = logits[..., allowed]
    for K in (4, 16, 20, 128):
        _check(beam_step(masked, scores, keep=K), masked, scores, None, None, K)
    start = torch.full((3, 4), -math.inf).cuda()
    start[:, 0] = 0
    step = beam_step(logits, start, keep=8)
    _check(step, logits, start, None, None, 8)
    assert (step.parents.cpu() == torch.arange(3)[:, None] * 4).all()
    masked[1, 2] = -math.inf  # a row without a token
    masked[0, 1, 5] = math.nan  # rows that hold a NaN, or +inf
    masked[0, 2, 77] = math.inf
    masked[2, :, 0] = math.nan
    scores[1, 0] = math.nan
    scores[1, 3] = math.inf
    _check(beam_step(masked, scores, keep=32), masked, scores, None, None, 32)
    dead = torch.full((1, 2, 5), math.nan).cuda()
    step = beam_step(dead, torch.zeros((1, 2)).cuda(), keep=7)
    assert (step.scores == -math.inf).all() and step.tokens[0].tolist() == [0, 1, 2, 3, 4, 0, 1] and step.parents[0].tolist() == [0] * 5 + [1] * 2


def test_finished_beams(gpu):
    """All finished; a finished beam's logits are not read; its rank keeps its own length."""
    logits, scores, lengths, _ = _inputs(8, 2, 5, 700, torch.float16)
    everyone = torch.ones((2, 5), dtype=torch.bool).cuda()
    step = beam_step(torch.full_like(logits, math.nan), scores, lengths, everyone, keep=5, pad=9, alpha=0.7)
    _check(step, logits, scores, lengths, everyone, 5, None, 9, 0.7)
    assert (step.tokens == 9).all() and step.finished.all()
    some = everyone.clone()
    some[:, ::2] = False
    bad = logits.clone()
    bad[some] = math.nan
    a, b = (beam_step(x, scores, lengths, some, keep=12, end=3, alpha=1.5) for x in (logits, bad))
    _check(a, logits, scores, lengths, some, 12, 3, None, 1.5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    _check(beam_step(logits, scores, lengths, some, keep=64, end=3), logits, scores, lengths, some, 64, 3)


@pytest.mark.parametrize("size", [1e-30, 1e4, 3e38])
def test_logits_of_every_size(gpu, size):
    logits, scores, _, _ = _inputs(3, 2, 3, 5000, torch.float32, spread=1.0)
    logits = logits.clamp(-1, 1) * size
    _check(beam_step(logits, scores, keep=8), logits, scores, None, None, 8)


def test_strides(gpu):
    big, scores, lengths, finished = _inputs(6, 4, 6, 2 * 999 + 3, torch.bfloat16, 0.2)
    part = big[1:3, ::2, 5:1004]
    wide = scores[1:3, ::2]
    want = beam_step(part.contiguous(), wide.contiguous(), keep=9)
    _check(want, part, wide, None, None, 9)
    assert all(torch.equal(a, b) for a, b in zip(beam_step(part, wide, keep=9), want) if a is not None)
    turned = part.transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(beam_step(turned, wide, keep=9), want) if a is not None)
    apart = big[1:3, ::2, 5:2003:2]
    _check(beam_step(apart, wide, keep=9), apart, wide, None, None, 9)
    row = big[1:3, :1, 5:1004].expand(2, 6, 999)
    _check(beam_step(row, scores[1:3], keep=9), row, scores[1:3], None, None, 9)


def test_rows_past_32_bits(gpu):
    """Logits of more than 2^32 elements: the last sequences are read where they lie."""
    V, W = 1 << 20, 2
    B = (1 << 32) // (V * W) + 3
    logits = torch.zeros((B, W, V), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    last = (torch.randn((2, W, V), generator=g) * 3).bfloat16().cuda()
    logits[-2:] = last
    scores = torch.zeros((B, W)).cuda()
    step = beam_step(logits, scores, keep=2)
    alone = beam_step(last, scores[-2:], keep=2)
    assert torch.equal(step.tokens[-2:], alone.tokens) and torch.equal(step.scores[-2:], alone.scores)
    assert torch.equal(step.parents[-2:], alone.parents + (B - 2) * W)
    assert (step.tokens[:-2].cpu() == torch.tensor([0, 1])).all()  # of the first of two like beams


def test_captured_and_another_stream(gpu):
    logits, scores, lengths, finished = _inputs(12, 4, 8, 30011, torch.bfloat16, 0.2)
    state = torch.randn((32, 100)).cuda()

    def step():
        s = beam_step(logits, scores, lengths, finished, end=5, alpha=0.5)
        return [*s, reorder(state, s.parents)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    g = torch.Generator().manual_seed(2)
    for i in range(4):
        if i:
            logits.copy_((torch.randn(logits.shape, generator=g) * 3).bfloat16())
            scores.copy_(-torch.rand(scores.shape, generator=g))
        want = step()
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("shape,dtype", [((7, 3, 5), torch.float32), ((9, 1024), torch.bfloat16), ((4, 13), torch.uint8),
                                         ((4, 7), torch.bool), ((6, 5), torch.int16), ((5,), torch.int64), ((3, 300001), torch.float16),
                                         ((2, 0), torch.float32), ((600, 2), torch.float64)])
def test_reorder(gpu, shape, dtype):
    g = torch.Generator().manual_seed(len(shape))
    state = torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=g).to(dtype).cuda()
    parents = torch.randint(0, shape[0], (3, 5), generator=g).cuda()
    want = state[parents.reshape(-1)]
    got = reorder(state, parents)
    assert got.dtype == dtype and torch.equal(got, want)
    pair = reorder([state, state], parents)
    assert len(pair) == 2 and torch.equal(pair[1], want)
    parents[0, 0], parents[2, 4] = -1, shape[0]
    want = want.clone()
    want[0], want[-1] = 0, 0
    assert torch.equal(reorder(state, parents), want)
    wide = torch.cat([state, state])[::2]  # rows apart
    ok = torch.arange(wide.shape[0]).cuda()
    assert torch.equal(reorder(wide, ok), wide)
    assert torch.equal(reorder(state.flip(0) if state.dim() == 1 else state.transpose(0, -1), ok[:1]),
                       (state.flip(0) if state.dim() == 1 else state.transpose(0, -1))[:1]) or state.numel() == 0
    assert reorder(state, parents[:0]).shape == (0, *shape[1:])


def test_nothing_to_do(gpu):
    step = beam_step(torch.empty((0, 3, 100)).cuda(), torch.empty((0, 3)).cuda(), keep=2)
    assert step.tokens.shape == (0, 2)


def test_refusals(gpu):
    logits, scores, lengths, finished = _inputs(1, 2, 3, 50, torch.float32)
    for bad in (dict(keep=0), dict(keep=129), dict(keep=151 - 300), dict(end=50), dict(pad=-1), dict(alpha=-0.5, lengths=lengths),
                dict(alpha=0.5), dict(alpha=math.nan, lengths=lengths), dict(alpha=math.inf, lengths=lengths),
                dict(finished=finished), dict(lengths=lengths.float()), dict(lengths=lengths[:1]),
                dict(finished=finished.int(), end=1), dict(finished=finished.cpu(), end=1)):
        with pytest.raises(ValueError):
            beam_step(logits, scores, **bad)
    for a, b in ((logits[0], scores), (logits.double(), scores), (logits, scores.half()), (logits, scores[:, :2]), (logits.cpu(), scores),
                 (logits, scores.cpu()), (logits[:, :, :0], scores)):
        with pytest.raises(ValueError):
            beam_step(a, b)
    with pytest.raises(ValueError):
        beam_step(torch.zeros((1, 129, 5)).cuda(), torch.zeros((1, 129)).cuda(), keep=3)
    with pytest.raises(ValueError):
        beam_step(torch.zeros((1, 1, 1 << 21), dtype=torch.bfloat16).cuda(), torch.zeros((1, 1)).cuda(), keep=128)
    with pytest.raises(RuntimeError, match="backward"):
        beam_step(logits.clone().requires_grad_(True), scores)
    with torch.no_grad():
        beam_step(logits.clone().requires_grad_(True), scores)
    parents = torch.zeros(2, dtype=torch.int64).cuda()
    for a, b in ((scores, parents.int()), (scores.cpu(), parents), (scores, parents.cpu()), (scores[0, 0], parents)):
        with pytest.raises(ValueError):
            reorder(a, b)
    with pytest.raises(RuntimeError, match="backward"):
        reorder(scores.clone().requires_grad_(True), parents)
