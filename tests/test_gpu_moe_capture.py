"""GPU tests of captured gradients of the norm's and the sparse layer's operators: what a capture can follow is taken
(a second stream that takes part in it, operands whose gradient nobody asks for), and a leaf that an eager graph
holds is refused however far behind the operator it lies."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F4 = torch.float32


def seeded(shape, seed, dtype=F4):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def operators():
    """name -> (operator of one operand, that operand's value)"""
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    x, w = seeded((12, 64), 1), seeded((64,), 2)
    order = moe_sort(moe_route(x[:, :8], 2)[1], 8)
    rows, weights = seeded((24, 64), 3), seeded((12, 2), 4)
    return {"rms_norm": (lambda t: rms_norm(t, w), x), "moe_route": (lambda t: moe_route(t, 2)[0], x),
            "moe_gather": (lambda t: moe_gather(t, order), x), "moe_combine": (lambda t: moe_combine(t, weights, order), rows)}


NAMES = ["rms_norm", "moe_route", "moe_gather", "moe_combine"]


def replays_equal(graph, got, want):
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_a_capture_that_forks_to_a_second_stream(cuda, name):
    op, value = operators()[name]

    def step(x, d, side):
        leaf = x.detach().requires_grad_(True)
        t = leaf * 2.0
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = op(t)
        torch.cuda.current_stream().wait_stream(side)
        return torch.autograd.grad(y, leaf, d)[0]

    d = torch.ones_like(op(value)) + torch.arange(op(value).shape[-1], device=cuda)
    want = step(value, d, torch.cuda.Stream())
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = step(value, d, side)
    replays_equal(graph, got, want)


def test_an_eagerly_held_operand_whose_gradient_nobody_asks_for(cuda):
    from stratum_amd import moe_combine, moe_route, moe_sort, rms_norm
    x, w, r = seeded((12, 64), 1), seeded((64,), 2).requires_grad_(True), seeded((12, 64), 3)
    order = moe_sort(moe_route(x[:, :8], 2)[1], 8)
    y, weights = seeded((24, 64), 4), seeded((12, 2), 5).requires_grad_(True)
    for op, held, value in ((lambda t: rms_norm(t, w), w, x), (lambda t: rms_norm(t, w, 1e-6, r)[0], w, x),
                            (lambda t: moe_combine(t, weights, order), weights, y)):
        leaf = value.clone().requires_grad_(True)
        d = torch.ones_like(op(value))
        want, = torch.autograd.grad(op(leaf), leaf, d)
        eager = op(value)  # a graph of the held operand alone
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(op(leaf), leaf, d)
        replays_equal(graph, got, want)
        assert torch.autograd.grad(eager, held, d)[0].isfinite().all()


@pytest.mark.parametrize("name", NAMES)
def test_an_eager_graphs_leaf_behind_other_operations_is_refused(cuda, name):
    op, value = operators()[name]
    leaf = value.clone().requires_grad_(True)
    eager = op(leaf)
    d = torch.ones_like(eager)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=f"{name}.*captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(op(leaf.view(-1).view(value.shape) * 1.0), leaf, d)
    torch.cuda.synchronize()
    assert torch.autograd.grad(eager, leaf, d)[0].isfinite().all()


def test_captured_gradients_that_accumulate(cuda):
    """backward() of leaves that no eager graph holds, through several of the operators."""
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    x, w, router = seeded((12, 64), 1), seeded((64,), 2), seeded((8, 64), 3)
    d = seeded((12, 64), 4)

    def step(x, w):
        y = rms_norm(x, w)
        weights, experts = moe_route(y @ router.t(), 2)
        order = moe_sort(experts, 8)
        moe_combine(moe_gather(y, order), weights, order, x).backward(d)

    want = [t.clone().requires_grad_(True) for t in (x, w)]
    step(*want)
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    for t in leaves:
        t.grad = torch.zeros_like(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*leaves)
    for i in range(3):
        for t in leaves:
            t.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, want))


@pytest.mark.parametrize("name", NAMES)
def test_a_leaf_of_an_eager_graph_on_a_stream_that_can_join(cuda, name):
    """Work on any but the null stream becomes part of a capture when it waits for it, as the engine makes it do."""
    op, value = operators()[name]
    leaf = value.clone().requires_grad_(True)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        eager = op(leaf)
        d = torch.ones_like(eager) + torch.arange(eager.shape[-1], device=cuda)
        want, = torch.autograd.grad(eager, leaf, d, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(op(leaf * 1.0), leaf, d)
    replays_equal(graph, got, want)
    assert torch.equal(torch.autograd.grad(eager, leaf, d)[0], want)
