"""GPU: beam steps and reorderings of more rows than one launch has room for (a launch's threads are fewer than 2^32)."""

import pytest
import torch

from ngram_amd.beam import beam_step, reorder

pytestmark = pytest.mark.gpu

LSE = 2.0**-20 + 2.0**-23 + 31 * 2.0**-24  # what a row's log-sum may be off by: test_beam_gpu.py derives it


@pytest.mark.parametrize("B,W,V,K,dtype", [((1 << 17) + 5, 128, 4, 2, torch.bfloat16), ((1 << 22) + 3, 4, 3, 1, torch.float32),
                                           (70001, 64, 70, 100, torch.float16)])
def test_steps_of_many_rows(gpu, B, W, V, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(W)
    logits = torch.randn((B, W, V), generator=g, device="cuda").to(dtype)
    scores = torch.randn((B, W), generator=g, device="cuda")
    lengths = torch.randint(0, 9, (B, W), generator=g, device="cuda").int()
    finished = torch.rand((B, W), generator=g, device="cuda") < 0.1
    step = beam_step(logits, scores, lengths, finished, keep=K, end=V - 1)
    assert ((step.parents // W) == torch.arange(B, device="cuda")[:, None]).all()
    at = step.parents % W * V + step.tokens
    order = at.sort(1).values
    assert ((order[:, 1:] > order[:, :-1]).all())  # no candidate twice
    for b0 in range(0, B, 1 << 17):
        b = slice(b0, min(B, b0 + (1 << 17)))
        total = logits[b].double().log_softmax(-1) + scores[b].double()[..., None]
        total.masked_fill_(finished[b][..., None], -float("inf"))
        total[..., V - 1] = torch.where(finished[b], scores[b].double(), total[..., V - 1])
        total = total.flatten(1)
        want, mine = total.topk(K, 1).values, total.gather(1, at[b])
        assert ((mine - want).abs() <= 2 * LSE).all()
        assert ((step.scores[b] - mine).abs() <= LSE + 2.0**-24 * mine.abs()).all()
    beam = step.parents % W
    done = finished.gather(1, beam)
    assert torch.equal(step.finished, done | (step.tokens == V - 1))
    assert torch.equal(step.lengths, lengths.gather(1, beam).long() + (~done).long())


def test_many_reordered_rows(gpu):
    g = torch.Generator(device="cuda").manual_seed(1)
    state = torch.randint(0, 1 << 30, (1000,), generator=g, device="cuda")
    parents = torch.randint(-1, 1001, ((1 << 24) + 12345,), generator=g, device="cuda")
    want = torch.where((parents >= 0) & (parents < 1000), state[parents.clamp(0, 999)], 0)
    assert torch.equal(reorder(state, parents), want)
    wide = state.view(10, 100)
    few = parents[:(1 << 22) + 7].clamp(0, 9)
    assert torch.equal(reorder(wide, few), wide[few])
