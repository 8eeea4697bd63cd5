"""GPU: the ranks of finished beams (ngram_amd.beam), which hold no log-sum: 64 bits from the exponent to the comparison."""

import pytest
import torch

from ngram_amd.beam import beam_step

pytestmark = pytest.mark.gpu


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


@pytest.mark.parametrize("alpha", [0.6, 0.1, 0.75, 1.0, 2.5])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_ranks_of_finished_beams(gpu, alpha, seed):
    """A finished beam's rank has no log-sum: its score over the power of its length, in 64 bits. Scores that tie within a
    float32's rounding come in the order of their ranks; the power, its quotient and the definition's are each off by an ulp of
    2^-52 at most, so ranks within 2^-50 of each other may come either way."""
    g = torch.Generator().manual_seed(seed)
    W = 128
    lengths = torch.randint(1, 2000, (1, W), generator=g)
    scores = (-384.0 * lengths.double() ** alpha).float()
    rank = [float(s) / n ** alpha for s, n in zip(scores[0].tolist(), lengths[0].tolist())]
    step = beam_step(torch.zeros((1, W, 5)).cuda(), scores.cuda(), lengths.cuda(), torch.ones((1, W), dtype=torch.bool).cuda(), end=2,
                     alpha=alpha)
    got = step.parents[0].tolist()
    want = sorted(range(W), key=lambda w: (-rank[w], w))
    assert sorted(got) == list(range(W))
    for a, b in zip(got, want):
        assert a == b or abs(rank[a] - rank[b]) <= 2.0**-50 * abs(rank[b]), (a, b, rank[a], rank[b])


def test_ranks_of_an_example(gpu):
    """Two finished beams, of 1 token and of 542: -384.025360 and -384.025382 with an exponent of 0.6 (in 32 bits it is
    0.60000002, and the second's -384.025325)."""
    scores = torch.tensor([[-16778.74609375, -384.02536]]).cuda()
    step = beam_step(torch.zeros((1, 2, 3)).cuda(), scores, _dev([[542, 1]]), torch.ones((1, 2), dtype=torch.bool).cuda(), end=0, alpha=0.6)
    assert step.parents.tolist() == [[1, 0]]


def test_equal_ranks_of_different_lengths(gpu):
    """Scores of -n over n tokens: all rank -1, and the lower beam comes first."""
    n = torch.randperm(128, generator=torch.Generator().manual_seed(4))[None] + 1
    step = beam_step(torch.zeros((1, 128, 3)).cuda(), -n.float().cuda(), n.cuda(), torch.ones((1, 128), dtype=torch.bool).cuda(), end=0,
                     alpha=1.0)
    assert step.parents[0].tolist() == list(range(128))
