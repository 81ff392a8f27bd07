"""Derivatives of the balance loss that are not a plain backward: forward mode, torch.func's transforms, batched
gradients, derivatives of derivatives.  On the CPU a stand-in takes the place of the kernels' launches, which tests
the rules around them; on the GPU the kernels run.

Tolerances: fp32 formulas of E <= 12 and T <= 12 terms, some 50 roundings of 2^-24 each on terms of the result's
size or, in sums, of the sum of absolute values: 1e-5 of the largest element.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

T, E, K = 11, 7, 2


def _exact(z, freq, mask):
    """The loss in the type of z, by the definition."""
    p = torch.softmax(z if mask is None else z.where(mask[:, None], torch.zeros_like(z)), -1)
    if mask is not None:
        p = p * mask[:, None]
    return E * (p.sum(0) / p.sum() * (freq / freq.sum())).sum()


def _raw(t):
    """The plain values behind a pointer: no tangent, and an error for a tensor without storage."""
    return torch.from_numpy(t.detach().numpy().copy())


def _stand_in(z, freq=None, idx=None, mask=None, err=None):
    with torch.no_grad():
        z, freq, idx, mask = (None if t is None else _raw(t) for t in (z, freq, idx, mask))
        on = torch.ones(len(z), dtype=torch.bool) if mask is None else mask
        if freq is None:
            freq = torch.nn.functional.one_hot(idx.long(), E)[on].sum((0, 1)).int()
        f, n = freq.double(), on.sum().double()
        coef = (E * f - f.sum()) / (f.sum() * n)
        return _exact(z.double(), f, mask).float(), freq.clone(), coef.float()


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def case(request, monkeypatch):
    from sonicmoe import functional as fn

    if request.param == "cpu":
        def bwd(z, coef, dloss, mask=None):
            z, coef, dloss, mask = (None if t is None else _raw(t) for t in (z, coef, dloss, mask))
            return (dloss * fn._switch_loss_gradient(z, coef, mask)).to(z.dtype)

        monkeypatch.setattr(fn.ops, "switch_loss", _stand_in)
        monkeypatch.setattr(fn.ops, "switch_loss_bwd", bwd)
    g = torch.Generator().manual_seed(3)
    z = torch.randn(T, E, generator=g).to(request.param)
    idx = torch.rand(T, E, generator=g).topk(K, 1).indices.int().to(request.param)
    mask = (torch.rand(T, generator=g) < 0.7).to(request.param)
    v = torch.randn(T, E, generator=g).to(request.param)
    freq = torch.nn.functional.one_hot(idx.long(), E)[mask].sum((0, 1))

    def loss(x):
        return fn.switch_load_balancing_loss(x, topk_indices=idx, token_mask=mask)[0]

    def exact(x):
        return _exact(x, freq.double(), mask)

    return fn, loss, exact, z, v


def _near(got, want):
    assert got.dtype == torch.float32 and got.shape == want.shape
    assert (got.double() - want).abs().max() <= 1e-5 * max(want.abs().max().item(), 1e-3)


@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode(case, needs_grad, recorded):
    fn, loss, exact, z, v = case
    _, want = torch.func.jvp(exact, (z.double(),), (v.double(),))
    with fwAD.dual_level(), torch.set_grad_enabled(recorded):
        out = fwAD.unpack_dual(loss(fwAD.make_dual(z.clone().requires_grad_(needs_grad), v)))
        assert out.tangent is not None
        _near(out.tangent.detach(), want)
        _near(out.primal.detach(), exact(z.double()))


def test_backward_of_forward_mode(case):
    fn, loss, exact, z, v = case
    want = torch.func.grad(lambda x: torch.func.jvp(exact, (x,), (v.double(),))[1])(z.double())
    leaf = z.clone().requires_grad_()
    with fwAD.dual_level():
        tangent = fwAD.unpack_dual(loss(fwAD.make_dual(leaf, v))).tangent
        (got,) = torch.autograd.grad(tangent, leaf)
    _near(got, want)


def test_forward_mode_through_the_backward(case):
    fn, loss, exact, z, v = case
    want = torch.func.jvp(torch.func.grad(exact), (z.double(),), (v.double(),))[1]
    with fwAD.dual_level():
        dual = fwAD.make_dual(z.clone().requires_grad_(), v)
        (g,) = torch.autograd.grad(loss(dual), dual)
        got = fwAD.unpack_dual(g).tangent
    assert got is not None
    _near(got, want)


def test_func_transforms(case):
    fn, loss, exact, z, v = case
    F = torch.func
    _near(F.grad(loss)(z), F.grad(exact)(z.double()))
    _near(F.jvp(loss, (z,), (v,))[1], F.jvp(exact, (z.double(),), (v.double(),))[1])
    _near(F.jacfwd(loss)(z), F.grad(exact)(z.double()))
    _near(F.hessian(loss)(z), F.hessian(exact)(z.double()))
    zs = torch.stack((z, v, z + v))
    _near(F.vmap(loss)(zs), F.vmap(exact)(zs.double()))
    _near(F.vmap(F.grad(loss))(zs), F.vmap(F.grad(exact))(zs.double()))
    _near(F.vmap(loss, in_dims=1)(zs.transpose(0, 1)), F.vmap(exact)(zs.double()))


def test_vmap_over_counts_and_masks(case):
    fn, _, _, z, v = case
    freqs = torch.arange(3 * E, device=z.device, dtype=torch.int32).reshape(3, E)
    masks = torch.arange(3 * T, device=z.device).reshape(3, T) % 4 != 1
    got, counts = torch.func.vmap(lambda f, m: fn.switch_load_balancing_loss(z, expert_frequency=f, token_mask=m))(
        freqs, masks)
    _near(got, torch.stack([_exact(z.double(), f.double(), m) for f, m in zip(freqs, masks)]))
    assert torch.equal(counts, freqs)


def test_batched_gradients(case):
    fn, loss, exact, z, v = case
    leaf = z.clone().requires_grad_()
    w = torch.tensor([1.0, -2.0, 0.5], device=z.device)
    (got,) = torch.autograd.grad(loss(leaf), leaf, w, is_grads_batched=True)
    _near(got, w[:, None, None] * torch.func.grad(exact)(z.double()))


def test_second_derivatives_by_autograd(case):
    fn, loss, exact, z, v = case
    leaf = z.clone().requires_grad_()
    _near(torch.autograd.functional.hessian(loss, leaf), torch.func.hessian(exact)(z.double()))
