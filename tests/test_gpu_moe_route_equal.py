"""GPU tests of the router's choice where different logits have one score in 64 bits (sigmoids that end at one or at zero,
softmax scores that do, values next to zero) and the scores are the keys: the lowest index, whichever of them the larger
logit is, for a token alone and beside others."""

import pytest
import torch

from test_gpu_moe import BF, F4, FP, choose

pytestmark = pytest.mark.gpu

LOW = [-5.0, -6.0, -7.0, -8.0]


def check(logits, k, score, groups, top_groups, dtype=F4):
    """The choice of all tokens at once, and of each alone."""
    from stratum_amd import moe_route
    logits = logits.to(dtype)
    how = dict(score=score, groups=groups, top_groups=top_groups, group_score="top2")
    want = choose(logits, k, **how)
    x = logits.cuda()
    for at in range(min(len(logits), 40)):
        one = moe_route(x[at:at + 1], k, **how)[1].cpu()
        assert torch.equal(one, want[at:at + 1]), (at, logits[at].tolist())
    together = moe_route(x, k, **how)[1].cpu()
    assert torch.equal(together, want)
    if logits.shape[1] <= 128:  # a token's neighbours in a wave, settled at once
        calm = torch.linspace(-3.0, 3.0, logits.shape[1], dtype=F4).to(dtype).expand(3, -1)
        beside = torch.cat([calm, logits[:1]]).cuda()
        assert torch.equal(moe_route(beside, k, **how)[1].cpu()[3:], want[:1])


@pytest.mark.parametrize("dtype", [F4, BF, FP])
@pytest.mark.parametrize("row,score,groups,top_groups,k", [
    # a smaller logit behind two equal ones has their score, and a lower index
    ([49.0, 50.0, 50.0, 49.5, *LOW], "sigmoid", 2, 1, 1),
    ([0.0, -801.0, -800.0, -800.0, -900.0, -901.0, -902.0, -903.0], "softmax", 2, 1, 2),
    ([-801.0, 0.0, -800.0, -800.0, -900.0, -901.0, -902.0, -903.0], "softmax", 2, 2, 3),
    ([-770.0, -760.0, -760.0, -765.0, -1000.0, -900.0, -800.0, -820.0], "sigmoid", 2, 2, 1),
    # a larger logit before two equal ones has their score, and a higher index
    ([0.0, 0.0, 0.0, 40.0, 0.0, 0.0, 0.0, 0.0, 0.0, 40.0, 0.0, 0.0, 0.0, 0.0, 0.0, 41.0], "sigmoid", 2, 2, 2),
    ([0.0, 0.0, 0.0, 40.0, 0.0, 0.0, 0.0, 40.0, 0.0, 40.0, 0.0, 0.0, 0.0, 0.0, 0.0, 41.0], "sigmoid", 2, 2, 3),
    # both
    ([48.0, 50.0, 50.0, 51.0, 50.0, 50.0, 48.0, 51.0], "sigmoid", 2, 2, 4),
    # equal logits alone, whose neighbours are apart
    ([1.0, 2.0, 2.0, 2.0, 2.0, 2.0, 2.0, 1.0], "sigmoid", 2, 2, 3),
    ([1.0, 2.0, 2.0, 2.0, 2.0, 2.0, 2.0, 1.0], "softmax", 2, 2, 5)])
def test_one_score_of_different_logits(cuda, row, score, groups, top_groups, k, dtype):
    check(torch.tensor([row]), k, score, groups, top_groups, dtype)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_logits_next_to_zero(cuda, score):
    """Differences that a score does not show."""
    for row in ([0.0, 1e-17, 1e-17, -1.0, *LOW], [0.0, 1e-17, 2e-17, 2e-17, -1.0, *LOW[:3]],
                [-1e-17, 0.0, 0.0, 1e-17, -1.0, *LOW[:3]]):
        for k in (1, 2, 3):
            check(torch.tensor([row]), k, score, 2, 1)


@pytest.mark.parametrize("E,groups,top_groups,k", [(8, 2, 1, 2), (16, 4, 3, 5), (16, 2, 2, 16), (60, 6, 4, 7), (128, 8, 4, 8),
                                                   (256, 8, 4, 8), (512, 16, 4, 10), (1024, 32, 6, 16)])
@pytest.mark.parametrize("score,values", [("sigmoid", [41.0, 42.0, 45.0, 50.0, -1.0, 3.0]),
                                          ("sigmoid", [-760.0, -770.0, -800.0, -1000.0]),
                                          ("softmax", [0.0, 1.0, -800.0, -801.0, -830.0, -900.0])])
def test_few_values(cuda, E, groups, top_groups, k, score, values):
    """Drawn from a handful of values, most of which share their score with others."""
    g = torch.Generator().manual_seed(E)
    logits = torch.tensor(values)[torch.randint(len(values), (24, E), generator=g)]
    check(logits, k, score, groups, top_groups)
    # few of them large: the choice ends among them, or right behind
    few = torch.where(torch.rand(24, E, generator=g) < 1.5 * k / E, logits, -20.0 - torch.arange(E) / 64)
    if score == "sigmoid" and values[0] > 0:
        check(few, k, score, groups, top_groups)
