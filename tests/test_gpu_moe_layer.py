"""GPU tests of the sparse layer's half as one run (NF4MoE), and of what its operators refuse there.

The layer rounds to bf16 where its operators meet (y, the logits, gate and up, their product, the experts' rows), as
the reference below does in 32 bits without those roundings; the bar is the one of the products on their own, 1e-2 of
the norm for bf16 and 5e-3 for fp16: six roundings of at most half a step, 2^-9 of a value as they spread, add up
to 2.4 of them (sqrt 6), 4.8e-3; two of them meet in the gating."""

import pytest
import torch

from gpu_checks import TOL

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32


def seeded(shape, seed, std=1.0, dtype=F4):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def layer(E=8, H=128, inter=64, k=2, dtype=BF, norm=True, **kw):
    from stratum_amd import NF4MoE, RMSNorm
    router = torch.nn.Linear(H, E, bias=False, device="cuda", dtype=dtype)
    with torch.no_grad():
        router.weight.copy_(seeded((E, H), 1, H ** -0.5 * 2))
    rms = RMSNorm(H, dtype=dtype, device="cuda") if norm else None
    gate_up, down = seeded((E, 2 * inter, H), 2, H ** -0.5, dtype), seeded((E, H, inter), 3, inter ** -0.5, dtype)
    return NF4MoE.quantize(router, gate_up, down, k, norm=rms, **kw)


def dense(moe, dtype):
    """The dequantized banks in 32 bits."""
    from stratum_amd import dequantize_4bit
    E, H, i, bs = moe.num_experts, moe.hidden, moe.inter, moe.blocksize
    return (dequantize_4bit(moe.gate_up_packed, absmax=moe.gate_up_absmax, blocksize=bs, dtype=dtype, shape=(E, 2 * i, H)).float(),
            dequantize_4bit(moe.down_packed, absmax=moe.down_absmax, blocksize=bs, dtype=dtype, shape=(E, H, i)).float())


def plain(moe, banks, x, residual, mask, chosen):
    """The layer in 32 bits with torch's gradients; the experts are given."""
    h = x if residual is None else x + residual
    y = h
    if moe.norm is not None:
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + moe.norm.eps) * moe.norm.weight.detach().float()
    else:
        y = x
    scores = torch.softmax(y @ moe.router.weight.detach().float().t(), -1)
    live = chosen >= 0
    w = torch.where(live, scores.gather(1, chosen.long().clamp(min=0)), 0.0)
    w = w / w.sum(1, keepdim=True).clamp_min(1e-20)
    out = residual if moe.norm is None else h
    out = torch.zeros_like(x) if out is None else out
    for e in range(moe.num_experts):
        gu = y @ banks[0][e].t()
        g, u = gu[:, :moe.inter], gu[:, moe.inter:]
        out = out + ((chosen == e) * w).sum(1, keepdim=True) * ((g * torch.sigmoid(g) * u) @ banks[1][e].t())
    return out


def close(got, want, dtype, what):
    off = ((got.float() - want).norm() / want.norm()).item()
    assert off <= TOL[dtype], f"{what}: {off}"


@pytest.mark.parametrize("tokens", [1, 2, 37, 300])
@pytest.mark.parametrize("dtype,stream,norm", [(BF, None, True), (BF, BF, True), (BF, F4, True), (FP, FP, True),
                                               (BF, BF, False), (BF, None, False)])
def test_the_layer_and_its_gradients(cuda, tokens, dtype, stream, norm):
    from stratum_amd import moe_route
    moe = layer(dtype=dtype, norm=norm, E=8 if tokens < 100 else 24)
    banks = dense(moe, dtype)
    x, r = seeded((tokens, 128), 5, 1.0, dtype), seeded((tokens, 128), 6, 1.0, stream) if stream else None
    mask = torch.ones(tokens, dtype=torch.bool, device=cuda)
    mask[3::5] = False
    with torch.no_grad():
        got = moe(x, r, mask)
        y = x if moe.norm is None else moe.norm(x) if r is None else moe.norm(x, r)[0]
        _, chosen = moe_route(moe.router(y), 2, mask=mask)
        wide = [t.float().requires_grad_(True) for t in (x, r) if t is not None]
    assert got.shape == x.shape and got.dtype == (stream or dtype)
    want = plain(moe, banks, wide[0], wide[1] if stream else None, mask, chosen)
    close(got, want.detach(), dtype, "out")
    leaves = [t.clone().requires_grad_(True) for t in (x, r) if t is not None]
    out = moe(leaves[0], leaves[1] if stream else None, mask)
    assert torch.equal(out, got)
    d = seeded((tokens, 128), 7, 1.0, got.dtype)
    params = [moe.router.weight] + ([moe.norm.weight] if norm else [])
    grads = torch.autograd.grad(out, leaves + params, d)
    want.backward(d.float())
    for name, leaf, g, ref in zip(("dx", "dresidual"), leaves, grads, wide):
        assert g.dtype == leaf.dtype
        close(g, ref.grad, dtype, name)
    assert all(g.isfinite().all() for g in grads)


def test_shapes_padding_and_no_tokens(cuda):
    moe = layer()
    x, r = seeded((2, 9, 128), 1, 1.0, BF), seeded((2, 9, 128), 2, 1.0, BF)
    mask = torch.ones(2, 9, dtype=torch.bool, device=cuda)
    mask[1, 4:] = False
    out = moe(x, r, mask)
    assert out.shape == x.shape
    assert torch.equal(out[1, 4:], moe.norm(x, r)[1][1, 4:])  # padding passes the stream on
    x2 = x.clone()
    x2[1, 4:] = float("nan")
    assert torch.equal(moe(x2, r, mask)[mask], out[mask])  # and what it holds matters to nobody
    nobody = torch.zeros(2, 9, dtype=torch.bool, device=cuda)
    assert torch.equal(moe(x, r, nobody), moe.norm(x, r)[1])
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(moe(leaf, r, nobody), leaf, x)
    assert torch.equal(g, x)
    assert moe(x[:, :0], r[:, :0]).shape == (2, 0, 128)


def test_sigmoid_scores_with_bias_and_groups(cuda):
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort
    bias = seeded((16,), 9, 0.1)
    kw = dict(score="sigmoid", groups=4, top_groups=2, group_score="top2", scale=2.5)
    moe = layer(E=16, k=4, bias=bias, **kw)
    x, r = seeded((50, 128), 1, 1.0, BF), seeded((50, 128), 2, 1.0, BF)
    out = moe(x, r)
    y, h = moe.norm(x, r)
    w, e = moe_route(moe.router(y), 4, bias=bias, **kw)
    order = moe_sort(e, 16)
    assert torch.equal(out, moe_combine(moe.experts(moe_gather(y, order), order), w, order, h))
    moe.to(BF)  # the bias is a buffer and is rounded with the others; it is used in 32 bits
    assert moe(x, r).isfinite().all()


def test_a_training_step_learns_nothing_it_should_not(cuda):
    """Only the router and the norm train; the banks stay as they are."""
    from stratum_amd import AdamW
    moe = layer()
    banks = [t.clone() for t in (moe.gate_up_packed, moe.gate_up_absmax, moe.down_packed, moe.down_absmax)]
    params = [p for p in moe.parameters() if p.requires_grad]
    assert len(params) == 2
    before = [p.detach().clone() for p in params]
    optimizer = AdamW(params, lr=1e-2)
    moe(seeded((40, 128), 1, 1.0, BF), seeded((40, 128), 2, 1.0, BF)).float().square().mean().backward()
    optimizer.step()
    assert all(not torch.equal(a, p.detach()) for a, p in zip(before, params))
    now = (moe.gate_up_packed, moe.gate_up_absmax, moe.down_packed, moe.down_absmax)
    assert all(torch.equal(a, b) for a, b in zip(banks, now))


def test_refusals(cuda):
    from stratum_amd import MoEOrder, moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    x, w = seeded((4, 16), 1, 1.0, BF), seeded((16,), 2, 1.0, BF)
    cpu = torch.ones(16, dtype=BF)
    e = torch.zeros(4, 2, dtype=torch.int32, device=cuda)
    order = moe_sort(e, 8)
    y, weights = seeded((8, 16), 3, 1.0, BF), seeded((4, 2), 4)
    o, s, p = order
    for call in (lambda: rms_norm(x, w[:8]), lambda: rms_norm(x, w.half()), lambda: rms_norm(x, cpu),
                 lambda: rms_norm(x, w, -1.0), lambda: rms_norm(x, w, 1e-6, x[:2]), lambda: rms_norm(x, w, 1e-6, x.half()),
                 lambda: rms_norm(x.double(), w.double()), lambda: rms_norm(x, w, 1e-6, x.cpu()),
                 lambda: rms_norm(x.float(), w), lambda: rms_norm(x[0, 0], w),
                 lambda: moe_route(x, 0), lambda: moe_route(x, 17), lambda: moe_route(x, -1), lambda: moe_route(x.double(), 2),
                 lambda: moe_route(seeded((4, 100), 1), 65), lambda: moe_route(seeded((4, 1025), 1), 2),
                 lambda: moe_route(x, 2, groups=3), lambda: moe_route(x, 2, groups=4, top_groups=5),
                 lambda: moe_route(x, 2, groups=0), lambda: moe_route(x, 3, groups=8, top_groups=1),
                 lambda: moe_route(x, 2, bias=w), lambda: moe_route(x, 2, bias=torch.zeros(8, device=cuda)),
                 lambda: moe_route(x, 2, bias=torch.zeros(16)), lambda: moe_route(x, 2, mask=torch.ones(4, device=cuda)),
                 lambda: moe_route(x, 2, mask=torch.ones(3, dtype=torch.bool, device=cuda)),
                 lambda: moe_sort(e.long(), 8), lambda: moe_sort(e, 0), lambda: moe_sort(e, 1025), lambda: moe_sort(e, -3),
                 lambda: moe_gather(x[:3], order), lambda: moe_gather(x[0], order), lambda: moe_gather(x.double(), order),
                 lambda: moe_gather(x, MoEOrder(o, s, p.long())), lambda: moe_gather(x, MoEOrder(o, s[:3], p)),
                 lambda: moe_gather(x, MoEOrder(o[:1], s, p)), lambda: moe_gather(x, MoEOrder(o.cpu(), s, p)),
                 lambda: moe_combine(y[None], weights, order), lambda: moe_combine(torch.cat([y, y]), weights, order),
                 lambda: moe_combine(y, weights.to(BF), order), lambda: moe_combine(y, weights[:2], order),
                 lambda: moe_combine(y, weights, order, x.half()), lambda: moe_combine(y, weights, order, x[:2]),
                 lambda: moe_combine(y, weights.cpu(), order), lambda: moe_combine(y.double(), weights, order)):
        with pytest.raises(ValueError):
            call()


def test_forward_mode_is_refused(cuda):
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    from torch.autograd import forward_ad
    x, w = seeded((4, 16), 1, 1.0, F4), seeded((16,), 2)
    order = moe_sort(torch.zeros(4, 2, dtype=torch.int32, device=cuda), 8)
    y, weights = seeded((8, 16), 3), seeded((4, 2), 4)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: rms_norm(dual(x), w), lambda: rms_norm(x, dual(w)), lambda: rms_norm(x, w, 1e-6, dual(x)),
                     lambda: moe_route(dual(x), 2), lambda: moe_gather(dual(x), order),
                     lambda: moe_combine(dual(y), weights, order), lambda: moe_combine(y, dual(weights), order),
                     lambda: moe_combine(y, weights, order, dual(x))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()


def test_a_changed_operand_is_noticed(cuda):
    """What a backward keeps must not have been written in the meantime."""
    from stratum_amd import rms_norm
    x, w = seeded((4, 16), 1).requires_grad_(True), seeded((16,), 2)
    leaf = x * 1.0
    y = rms_norm(leaf, w)
    with torch.no_grad():
        leaf.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_are_differentiable_once(cuda):
    """With create_graph the gradients are there and raise when they are differentiated."""
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    x, w, r = (seeded(s, i).requires_grad_(True) for i, s in enumerate(((4, 16), (16,), (4, 16))))
    order = moe_sort(torch.arange(8, dtype=torch.int32, device=cuda).view(4, 2) % 5, 5)
    y, weights = seeded((8, 16), 3).requires_grad_(True), seeded((4, 2), 4).requires_grad_(True)
    for call, leaves in ((lambda: rms_norm(x, w), (x, w)), (lambda: rms_norm(x, w, 1e-6, r)[0], (x, w, r)),
                         (lambda: rms_norm(x, w, 1e-6, r)[0], (r,)), (lambda: moe_route(x, 2)[0], (x,)),
                         (lambda: moe_gather(x, order), (x,)), (lambda: moe_combine(y, weights, order), (y, weights)),
                         (lambda: moe_combine(y, weights, order, r), (weights, r))):
        d = torch.ones_like(call())
        plain = torch.autograd.grad(call(), leaves, d)
        grads = torch.autograd.grad(call(), leaves, d, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        with pytest.raises(RuntimeError, match="differentiable once"):
            grads[0].sum().backward()


def test_tensor_subclasses(cuda):
    """Operands of a subclass give the results and gradients of their plain tensors."""
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm

    class Named(torch.Tensor):
        pass

    x, w, r = seeded((4, 16), 1), seeded((16,), 2), seeded((4, 16), 3)
    weights, e = moe_route(x, 2)
    order = moe_sort(e, 16)
    y = seeded((8, 16), 4)
    for call, args in ((lambda x, w, r: rms_norm(x, w, 1e-6, r)[0], (x, w, r)), (lambda x: moe_route(x, 2)[0], (x,)),
                       (lambda x: moe_gather(x, order), (x,)),
                       (lambda y, w, r: moe_combine(y, w, order, r), (y, weights, r))):
        results = []
        for kind in (torch.Tensor, Named):
            leaves = [t.detach().clone().as_subclass(kind).requires_grad_(True) for t in args]
            out = call(*leaves)
            grads = torch.autograd.grad(out, leaves, torch.ones(out.shape, device=cuda))
            results.append([torch.Tensor(t.detach()) for t in (out, *grads)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
    assert all(torch.equal(a, b) for a, b in zip(moe_sort(e.as_subclass(Named), 16), order))


def test_a_captured_gradient_of_an_eager_graphs_leaf_is_refused(cuda):
    """The engine cannot pass a gradient on from a capture to a leaf that an eager graph ties to another stream."""
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    x, w = seeded((12, 64), 1), seeded((64,), 2)
    order = moe_sort(moe_route(x[:, :8], 2)[1], 8)
    rows, weights = seeded((24, 64), 3), seeded((12, 2), 4)
    for name, op, operand in (("rms_norm", lambda t: rms_norm(t, w), x), ("moe_route", lambda t: moe_route(t, 2)[0], x),
                              ("moe_gather", lambda t: moe_gather(t, order), x),
                              ("moe_combine", lambda t: moe_combine(t, weights, order), rows)):
        leaf = operand.clone().requires_grad_(True)
        eager = op(leaf)
        d = torch.ones_like(eager)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=f"{name}.*captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(op(leaf), leaf, d)
        torch.cuda.synchronize()
        want, = torch.autograd.grad(eager, leaf, d)
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(op(leaf), leaf, d)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


def test_no_columns(cuda):
    from stratum_amd import moe_combine, moe_gather, moe_sort
    order = moe_sort(torch.tensor([[0, 1], [2, 0]], dtype=torch.int32, device=cuda), 4)
    y, w = torch.zeros(4, 0, dtype=BF, device=cuda, requires_grad=True), seeded((2, 2), 1).requires_grad_(True)
    out = moe_combine(y, w, order)
    assert out.shape == (2, 0)
    dy, dw = torch.autograd.grad(out, (y, w), torch.zeros_like(out))
    assert dy.shape == (4, 0) and torch.equal(dw, torch.zeros_like(w))
    assert moe_gather(torch.zeros(2, 0, dtype=BF, device=cuda), order).shape == (4, 0)
