"""GPU tests of the router's choice where keys lie nearer to each other than a 32-bit rounding: the experts are those of
the 64-bit keys, whichever way the kernel takes to them, and a token's do not depend on the tokens beside it."""

import pytest
import torch

from test_gpu_moe import BF, F4, check_route, choose, seeded

pytestmark = pytest.mark.gpu


def level(logits, score, at, experts):
    """A bias that brings the scores of *experts* of row 0 to *at*, as near as fp32 can."""
    s = (torch.softmax(logits[0].double(), 0) if score == "softmax" else torch.sigmoid(logits[0].double()))
    bias = torch.zeros(logits.shape[1], dtype=torch.float64)
    bias[experts] = at - s[experts]
    return bias.float()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(8, 3), (16, 16), (60, 4), (64, 20), (128, 8), (256, 8), (300, 40), (512, 8), (1024, 10)])
@pytest.mark.parametrize("share", [0.1, 1.0])
def test_many_nearly_equal_keys(cuda, E, k, score, share):
    """At share 1 there are more of them than a token has lanes."""
    logits = seeded((5, E), E, 1.5)
    few = torch.arange(E)[::max(1, round(1 / share))]
    check_route(logits, k, score=score, bias=level(logits, score, 2.0, few))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("E,groups,top_groups,k", [(16, 4, 2, 3), (60, 6, 2, 5), (128, 8, 4, 8), (256, 8, 4, 8), (512, 64, 9, 9)])
def test_nearly_equal_groups(cuda, E, groups, top_groups, k, score, group_score):
    logits = seeded((5, E), E, 1.5)
    two = torch.arange(E).view(groups, -1)[:, :2].reshape(-1)
    check_route(logits, k, score=score, bias=level(logits, score, 2.0, two), groups=groups, top_groups=top_groups,
                group_score=group_score)


def test_groups_whose_two_best_cancel(cuda):
    """Sums that are small beside their terms: 4 + small and -4 + small."""
    E, groups = 64, 8
    logits = seeded((7, E), 3, 1.0)
    bias = torch.full((groups, E // groups), -20.0)
    bias[:, 1], bias[:, 4] = 4.0, -4.0
    check_route(logits, 2, score="sigmoid", bias=bias.reshape(-1), groups=groups, top_groups=2, group_score="top2")


@pytest.mark.parametrize("dtype", [BF, F4])
@pytest.mark.parametrize("score,shift", [("sigmoid", 45.0), ("sigmoid", -720.0), ("softmax", 0.0)])
def test_scores_that_end(cuda, dtype, score, shift):
    """Different logits whose 64-bit scores are equal: the lowest index, not the larger logit. (The choice alone: where
    sigmoids end their share of each other is 0 / 0 in 64 bits.)"""
    from stratum_amd import moe_route
    logits = (seeded((4, 64), 9, 2.0) + shift).to(dtype)
    if score == "softmax":
        logits[:, ::8] += 1200.0
    how = dict(score=score, groups=4, top_groups=2, group_score="top2")
    _, experts = moe_route(logits.cuda(), 6, **how)
    assert torch.equal(experts.cpu(), choose(logits, 6, **how))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(16, 4), (64, 6), (128, 8), (256, 8)])
def test_a_large_batch_and_each_of_its_tokens(cuda, E, k, score):
    """Among many tokens some have near keys by chance."""
    from stratum_amd import moe_route
    logits, bias = seeded((30000, E), E, 1.5), seeded((E,), 1, 0.1)
    s = torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double())
    want = (s + bias.double()).sort(dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
    x = logits.cuda()
    _, experts = moe_route(x, k, score=score, bias=bias.cuda())
    assert torch.equal(experts.cpu(), want)
    for at in (0, 777, 29999):
        _, one = moe_route(x[at:at + 1], k, score=score, bias=bias.cuda())
        assert torch.equal(one.cpu(), want[at:at + 1])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_tokens_beside_one_with_near_keys(cuda, score):
    from stratum_amd import moe_route
    logits = seeded((64, 32), 5, 1.5)
    bias = level(logits, score, 1.0, torch.arange(32))
    want = choose(logits, 5, score, bias)
    _, experts = moe_route(logits.cuda(), 5, score=score, bias=bias.cuda())
    assert torch.equal(experts.cpu(), want)
    _, alone = moe_route(logits[1:].cuda(), 5, score=score, bias=bias.cuda())
    assert torch.equal(alone.cpu(), want[1:])
    bad = logits.clone()
    bad[0, 3] = float("nan")
    _, beside = moe_route(bad.cuda(), 5, score=score, bias=bias.cuda())
    assert torch.equal(beside.cpu()[1:], want[1:])


def test_infinite_biases(cuda):
    """An expert that is always chosen, one that never is."""
    from stratum_amd import moe_route
    logits, bias = seeded((40, 64), 2, 1.5), seeded((64,), 3, 0.1)
    bias[7], bias[20] = float("inf"), float("-inf")
    _, experts = moe_route(logits.cuda(), 6, score="sigmoid", bias=bias.cuda())
    assert torch.equal(experts.cpu(), choose(logits, 6, "sigmoid", bias))
    assert (experts[:, 0] == 7).all() and not (experts == 20).any()
