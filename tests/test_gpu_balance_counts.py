"""GPU tests of the balance loss on counts of other types than int32: loss and gradient against float64.

Tolerances: those of tests/test_gpu_balance.py, plus one rounding each of a count and of 1 / F to fp32 (2^-23 in the
loss, of max |c| in the gradient), which its 2.5e-5 and 3e-5 have room for.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fn():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import functional

    return functional


def _exact(z, f, mask):
    p = torch.softmax(z.double(), 1)
    if mask is not None:
        p = p * mask[:, None]
    n, f, E = p.sum(), f.double(), z.shape[1]
    c = E * f / (f.sum() * n)
    return E * (p.sum(0) / n * f / f.sum()).sum(), p * (c - (p * c).sum(1, keepdim=True)), \
        p * (E * f / f.sum() - 1).abs().max() / n


def _case(T, E):
    g = torch.Generator().manual_seed(T + E)
    z = torch.randn(T, E, generator=g).cuda()
    f = torch.randint(0, 1 + 8 * T, (E,), generator=g).cuda()
    f[0] += 1
    return z, f, (torch.rand(T, generator=g) < 0.7).cuda() if T > 1 else None


KINDS = {
    "fractions": lambda f: (f.double() / f.sum()).float(),
    "averages": lambda f: f.double() / 7,
    "half fractions": lambda f: (f.double() / f.sum()).half(),
    "small": lambda f: (f.double() / f.sum() * 1e-20).float(),
    "int64": lambda f: f,
    "int64 beyond int32": lambda f: f << 36,
    "int16": lambda f: (f % 30000).to(torch.int16),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E", [(1, 1), (5, 7), (40, 128), (9000, 12), (3000, 300), (70, 4096)])
def test_loss_and_gradient(fn, T, E, kind):
    z, f, mask = _case(T, E)
    f = KINDS[kind](f)
    if f.double().sum() == 0:
        f[0] = 1
    leaf = z.clone().requires_grad_()
    loss, back = fn.switch_load_balancing_loss(leaf, expert_frequency=f, token_mask=mask)
    (dl,) = torch.autograd.grad(loss, leaf)
    want, grad, bound = _exact(z, f, mask)
    assert torch.equal(back.double(), f.double())
    assert abs(loss.item() - want.item()) <= 2.5e-5 * want.item()
    assert ((dl.double() - grad).abs() <= 2.0 ** -24 * grad.abs() + 3e-5 * bound + 2.0 ** -126).all()


@pytest.mark.parametrize("T,E", [(5, 7), (9000, 12), (3000, 300)])
def test_whole_counts_give_the_same_bits_in_every_type(fn, T, E):
    z, f, mask = _case(T, E)
    want = fn.ops.switch_loss(z, f.int(), token_mask=mask)
    for dtype in (torch.int64, torch.float32, torch.float64):
        got = fn.ops.switch_loss(z, f.to(dtype), token_mask=mask)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and got[1].dtype == dtype
    got = fn.ops.switch_loss(z, f * 2.0 ** -40, token_mask=mask)  # proportions decide
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_traced(fn):
    z, f, mask = _case(500, 24)
    f = (f / f.sum()).float()

    def loss(x):
        return fn.switch_load_balancing_loss(x, expert_frequency=f, token_mask=mask)

    leaf = z.clone().requires_grad_()
    a, fa = torch.compile(loss, fullgraph=True)(leaf)
    (ga,) = torch.autograd.grad(a, leaf)
    b, fb = loss(leaf)
    (gb,) = torch.autograd.grad(b, leaf)
    assert torch.equal(a, b) and torch.equal(fa, fb) and torch.equal(ga, gb)


def test_nothing_counts(fn):
    z, f, _ = _case(40, 24)
    leaf = z.clone().requires_grad_()
    loss, _ = fn.switch_load_balancing_loss(leaf, expert_frequency=torch.zeros(24, device="cuda"))
    (dl,) = torch.autograd.grad(loss, leaf)
    assert loss.item() == 0.0 and (dl == 0).all()
