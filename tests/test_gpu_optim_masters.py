"""GPU tests of parameters that something else writes between two steps of an optimizer with fp32
masters. A first step with a constant gradient moves every element by lr (the moments' corrections
cancel), give or take 2^-20 of it; bf16 keeps 8 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(value, n=700, lr=2.0 ** -10, bits=32, dtype=torch.bfloat16):
    from stratum_amd.optim import AdamW
    p = torch.nn.Parameter(torch.full((n,), value, dtype=dtype, device="cuda"))
    opt = AdamW([p], lr=lr, weight_decay=0.0, state_bits=bits, master_weights=True)
    return p, opt


def step(p, opt):
    p.grad = torch.ones_like(p)
    opt.step()


def overwrite(p, how, value):
    if how == "data":
        p.data.fill_(value)
    elif how == "in place":
        with torch.no_grad():
            p.fill_(value)
    else:
        p.data = torch.full_like(p.data, value)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["data", "in place", "replaced"])
def test_a_written_parameter_is_taken_over(cuda, how, bits, dtype):
    p, opt = make(1.0, bits=bits, dtype=dtype)
    step(p, opt)
    overwrite(p, how, 3.0)
    step(p, opt)
    master = opt.state[p]["master"]
    assert (master < 3.0).all() and (master > 3.0 - 1.5 * 2.0 ** -10).all()
    assert torch.equal(p.data, master.to(dtype))


@pytest.mark.parametrize("how", ["data", "in place", "replaced"])
def test_a_write_between_load_and_step_is_taken_over(cuda, how):
    p, opt = make(1.0)
    step(p, opt)
    q, again = make(1.0)
    again.load_state_dict(opt.state_dict())
    overwrite(q, how, 3.0)
    step(q, again)
    assert (again.state[q]["master"] > 2.99).all() and (q > 2.9).all()


def test_only_the_written_elements_leave_their_masters(cuda):
    """The others keep what 16 bits round away, also through a copy of equal values over them."""
    n = 5000
    p, opt = make(1.0, n=n, lr=2.0 ** -14)  # 2^-14 is nothing to a bf16 one
    step(p, opt)
    before = opt.state[p]["master"].clone()
    assert (before < 1.0).all() and (p == 1.0).all()
    p.data[77] = -2.0
    p.data[n - 1] = float("inf")
    p.data.copy_(p.data.clone())
    step(p, opt)
    master = opt.state[p]["master"]
    written = torch.zeros(n, dtype=torch.bool, device=cuda)
    written[77] = written[n - 1] = True
    assert (master[~written] < before[~written]).all()
    assert (master[~written] > 1.0 - 3 * 2.0 ** -14).all()
    assert master[77].item() == pytest.approx(-2.0 - 2.0 ** -14, abs=2.0 ** -20) and master[n - 1].item() == float("inf")


@pytest.mark.parametrize("count", [3, 60])
def test_tensors_take_their_masters_unless_asked_to_follow(cuda, count):
    """Both forms of the list, sizes that end inside a tile, and bases between the aligned ones."""
    from stratum_amd.optim import AdamWTensors
    for follow in (False, True):
        ps = [torch.full((700 + 37 * i + 1,), 3.0, dtype=torch.bfloat16, device=cuda)[i % 2:] for i in range(count)]
        masters = [torch.ones(p.numel(), device=cuda) for p in ps]
        m, v = ([torch.zeros(p.numel(), device=cuda) for p in ps] for _ in range(2))
        AdamWTensors(ps, m, v, masters=masters, follow=follow).step([torch.ones_like(p) for p in ps], step=1, lr=0.25,
                                                                    weight_decay=0.0)
        want = 2.75 if follow else 0.75
        assert all(torch.allclose(x, torch.full_like(x, want), rtol=1e-6) for x in masters)
        assert all((p == want).all() for p in ps)


def test_following_changes_no_bit_where_nothing_was_written(cuda):
    from stratum_amd.optim import AdamWTensors
    results = []
    for follow in (False, True):
        g = torch.Generator().manual_seed(4)
        masters = [(torch.randn(n, generator=g) * 10.0 ** (n % 7 - 3)).to(cuda) for n in (1, 255, 4097, 70_001)]
        ps = [x.to(torch.float16) for x in masters]
        m, v = ([torch.zeros_like(x) for x in masters] for _ in range(2))
        tensors = AdamWTensors(ps, m, v, masters=masters, follow=follow)
        for t in range(1, 5):
            tensors.step([torch.randn(x.numel(), generator=g).to(cuda) for x in masters], step=t, lr=1e-3)
        results.append(ps + masters + m + v)
    assert all(torch.equal(a, b) for a, b in zip(*results))
