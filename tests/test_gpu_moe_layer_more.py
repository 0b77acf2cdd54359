"""GPU tests of the sparse layer as a module: its bias under conversions, the gradients of its parameters by value, and
recomputation."""

import copy

import pytest
import torch

from test_gpu_moe_layer import BF, F4, FP, close, dense, layer, seeded

pytestmark = pytest.mark.gpu


def test_the_bias_stays_in_32_bits(cuda):
    """A balancing bias tells keys apart that a 16-bit one does not."""
    bias = 1.0 + torch.arange(16, device=cuda) * 2.0 ** -12  # all of them 1 in bf16, and 2^-10 apart in fp16
    kw = dict(E=16, k=4, score="sigmoid")
    moe = layer(bias=bias, **kw)
    with torch.no_grad():
        moe.router.weight.zero_()  # the bias alone decides
    x, r = seeded((5, 128), 1, 1.0, BF), seeded((5, 128), 2, 1.0, BF)
    want = moe(x, r)
    for change in (lambda m: m.to(BF), lambda m: m.half().bfloat16(), lambda m: torch.nn.Sequential(m).to(BF)[0],
                   lambda m: m.to("cpu", BF).to(cuda), lambda m: copy.deepcopy(m).bfloat16(), lambda m: m.float().to(BF)):
        again = change(copy.deepcopy(moe))
        assert again.bias.dtype == F4 and torch.equal(again.bias, bias) and again.bias.device == bias.device
        assert "bias" in again.state_dict() and not again.bias.requires_grad
        assert torch.equal(again(x, r), want)
    moe.load_state_dict({n: t.to(BF) for n, t in moe.state_dict().items()})
    assert moe.bias.dtype == F4


def plain(moe, banks, x, residual, mask, chosen, router, weight):
    """The layer in 32 bits, with torch's gradients for the router's and the norm's weight too."""
    h = x if residual is None else x + residual
    y = x
    if weight is not None:
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + moe.norm.eps) * weight
    live = chosen >= 0
    scores = torch.softmax(y @ router.t(), -1)
    w = torch.where(live, scores.gather(1, chosen.long().clamp(min=0)), 0.0)
    w = w / w.sum(1, keepdim=True).clamp_min(1e-20)
    out = residual if weight is None else h
    out = torch.zeros_like(x) if out is None else out
    for e in range(moe.num_experts):
        g, u = (y @ banks[0][e].t()).split(moe.inter, 1)
        out = out + ((chosen == e) * w).sum(1, keepdim=True) * ((g * torch.sigmoid(g) * u) @ banks[1][e].t())
    return out


@pytest.mark.parametrize("tokens,E,k", [(37, 8, 2), (300, 24, 4), (300, 8, 3)])
@pytest.mark.parametrize("dtype,stream,norm", [(BF, None, True), (BF, BF, True), (BF, F4, True), (FP, FP, True),
                                               (FP, None, False)])
def test_the_gradients_of_its_parameters(cuda, tokens, E, k, dtype, stream, norm):
    """The bar of the layer's other gradients: to the six roundings on the way to the experts' rows come those of dout's
    product with them, the logits' gradient and the sum over tokens, nine of half a step in all, 3 * 2^-9 as they
    spread (bf16), and what the logits' own rounding moves the scores by, 2^-9 of about 2, as they spread."""
    from stratum_amd import moe_route
    moe = layer(dtype=dtype, norm=norm, E=E, k=k)
    banks = dense(moe, dtype)
    x, r = seeded((tokens, 128), 5, 1.0, dtype), seeded((tokens, 128), 6, 1.0, stream) if stream else None
    mask = torch.ones(tokens, dtype=torch.bool, device=cuda)
    mask[3::5] = False
    with torch.no_grad():
        y = x if not norm else moe.norm(x) if r is None else moe.norm(x, r)[0]
        _, chosen = moe_route(moe.router(y), k, mask=mask)
    params = [moe.router.weight] + ([moe.norm.weight] if norm else [])
    wide = [p.detach().float().requires_grad_(True) for p in params]
    d = seeded((tokens, 128), 7, 1.0, stream or dtype)
    grads = torch.autograd.grad(moe(x, r, mask), params, d)
    plain(moe, banks, x.float(), r.float() if stream else None, mask, chosen, wide[0],
          wide[1] if norm else None).backward(d.float())
    for name, p, got, ref in zip(("router", "norm"), params, grads, wide):
        assert got.dtype == p.dtype
        close(got, ref.grad, dtype, name)


def test_recomputation_gives_the_same_gradients(cuda):
    from torch.utils.checkpoint import checkpoint
    moe = layer(E=16, k=4)
    x, r = seeded((50, 128), 1, 1.0, BF), seeded((50, 128), 2, 1.0, BF)
    d = seeded((50, 128), 3, 1.0, BF)
    results = []
    for run in (moe, lambda a, b: checkpoint(moe, a, b, use_reentrant=False), lambda a, b: checkpoint(moe, a, b, use_reentrant=True)):
        leaves = [t.clone().requires_grad_(True) for t in (x, r)]
        moe.zero_grad()
        out = run(*leaves)
        out.backward(d)
        results.append([out.detach(), *(t.grad for t in leaves), *(p.grad.clone() for p in moe.parameters())])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_one_tensor_in_two_places(cuda):
    """x as its own residual, the experts' rows' weights of one tensor, one leaf for both: gradients add up."""
    from stratum_amd import moe_combine, moe_sort, rms_norm
    x, w = seeded((6, 96), 1, 1.0, F4), seeded((96,), 2)
    dy, dh = seeded((6, 96), 3), seeded((6, 96), 4)
    a = x.clone().requires_grad_(True)
    both, = torch.autograd.grad(rms_norm(a, w, 1e-6, a), a, (dy, dh))
    b, c = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    one, two = torch.autograd.grad(rms_norm(b, w, 1e-6, c), (b, c), (dy, dh))
    assert torch.equal(both, one + two)
    a.grad = None
    sum(t.mul(g).sum() for t, g in zip(rms_norm(a, w, 1e-6, a), (dy, dh))).backward()
    assert torch.equal(a.grad, both)
    order = moe_sort(torch.arange(6, dtype=torch.int32, device=cuda).view(6, 1), 6)
    weights = seeded((6, 1), 5)
    y = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(moe_combine(y, weights, order, y), y, dy)
    assert torch.equal(got, dy * weights + dy)


def test_a_batched_call_of_vmap_is_refused(cuda):
    from stratum_amd import moe_route, rms_norm
    x, w = seeded((3, 4, 16), 1), seeded((16,), 2)
    for call in (lambda t: rms_norm(t, w), lambda t: moe_route(t, 2)[0]):
        with pytest.raises(RuntimeError):
            torch.vmap(call)(x)
