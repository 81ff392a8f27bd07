"""GPU tests of the switch balance loss: loss, per-expert counts and gradient against float64.

Tolerances.  p = 2^t / sum with t = (x - max) log2 e: two roundings of t (|t| <= 45 here: 45 * 2^-23 * ln 2
< 4e-6), 2^-22 of the exponential, at most 40 roundings in the row's sum and quotient (40 * 2^-24): p is
within 1e-5 of itself.  The columns' sums add at most 200 roundings one after the other (1.2e-5).  The
loss, a mean of p with positive weights, is within 2.5e-5 of itself.  The gradient g p (c - mean) carries
p's 1e-5 and the mean's (1e-5 + 3 * 2^-24) of |c|: at most 3e-5 of g p max |c|, plus half a step of the
output type, eps / 2 of the value and half its smallest step.
"""
import pytest
import torch

from oracle import balance as obalance

pytestmark = pytest.mark.gpu

RTOL = 2.5e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def fn():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import functional

    return functional


def _case(T, E, K, dtype, seed, masked):
    g = torch.Generator().manual_seed(seed)
    z = (1.5 * torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)).to(dtype)
    idx = torch.rand(T, E, generator=g).topk(K, 1).indices.to(torch.int32)
    mask = torch.rand(T, generator=g) < 0.7 if masked else None
    return z.cuda(), idx.cuda(), None if mask is None else mask.cuda()


def _check(loss, freq, dl, z, ref, dtype):
    rloss, rfreq, rdl, bound = ref
    assert loss.dtype == torch.float32 and loss.shape == () and freq.dtype == torch.int32 and dl.dtype == dtype
    assert torch.equal(freq.long(), rfreq)
    assert abs(loss.item() - rloss.item()) <= RTOL * abs(rloss.item())
    step = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[dtype]
    # products below the smallest normal fp32 number may lose all their bits
    tol = torch.finfo(dtype).eps / 2 * rdl.abs() + 3e-5 * bound + step + 2.0 ** -126
    assert ((dl.double() - rdl).abs() <= tol).all()


SHAPES = [
    # T, E, K
    (1, 1, 1), (1, 8, 2), (3, 7, 3), (64, 128, 8), (257, 60, 6), (1000, 33, 4), (129, 256, 8), (77, 300, 5),
    (50, 1000, 8), (19, 1027, 8), (40, 4096, 8), (40000, 128, 8), (30011, 12, 2), (5000, 100, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,K", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_loss_counts_and_gradient(fn, T, E, K, dtype, masked):
    z, idx, mask = _case(T, E, K, dtype, T + E, masked)
    dloss = 0.37 * T if dtype == torch.float16 else 0.37  # keeps fp16 gradients in range
    ref = obalance.switch_loss(z, idx=idx, mask=mask, dloss=torch.tensor(dloss, dtype=torch.float32).item())
    leaf = z.clone().requires_grad_()
    loss, freq = fn.switch_load_balancing_loss(leaf, topk_indices=idx, token_mask=mask)
    (dl,) = torch.autograd.grad(loss, leaf, torch.tensor(dloss, device="cuda"))
    _check(loss.detach(), freq, dl, z, ref, dtype)
    # counts as given
    leaf2 = z.clone().requires_grad_()
    loss2, freq2 = fn.switch_load_balancing_loss(leaf2, expert_frequency=ref[1].int().cuda(), token_mask=mask)
    (dl2,) = torch.autograd.grad(loss2, leaf2, torch.tensor(dloss, device="cuda"))
    assert torch.equal(loss, loss2) and torch.equal(dl, dl2) and torch.equal(freq2.long(), ref[1])


@pytest.mark.parametrize("E", [6, 128, 2000])
def test_same_bits_every_time(fn, E):
    z, idx, _ = _case(9000, E, 4, torch.bfloat16, 5, False)
    a = fn.ops.switch_loss(z, topk_indices=idx)
    for _ in range(5):
        b = fn.ops.switch_loss(z, topk_indices=idx)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_masked_rows_are_not_looked_at(fn):
    z, idx, mask = _case(300, 40, 4, torch.bfloat16, 3, True)
    ref = fn.ops.switch_loss(z, topk_indices=idx, token_mask=mask)
    poisoned, ids = z.clone(), idx.clone()
    poisoned[~mask] = float("nan")
    poisoned[(~mask).nonzero()[::2, 0]] = float("inf")
    ids[~mask] = 1 << 30
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = fn.ops.switch_loss(poisoned, topk_indices=ids, token_mask=mask, err=err)
    assert all(torch.equal(a, b) for a, b in zip(ref, got)) and err.item() == 0
    dl = fn.ops.switch_loss_bwd(poisoned, got[2], torch.ones((), device="cuda"), mask)
    assert torch.equal(dl, fn.ops.switch_loss_bwd(z, got[2], torch.ones((), device="cuda"), mask))
    assert (dl[~mask] == 0).all()


@pytest.mark.parametrize("E", [16, 100, 1500])
def test_rows_with_infinities(fn, E):
    """-inf logits take no part, lowest-value rows are uniform, and a row without a finite maximum makes
    the loss NaN, as its softmax is."""
    z, idx, _ = _case(200, E, 4, torch.float32, 4, False)
    z[:, ::3] = -float("inf")
    z[7] = torch.finfo(torch.float32).min
    z[8, 1:] = torch.finfo(torch.float32).min
    ref = obalance.switch_loss(z, idx=idx, dloss=1.0)
    leaf = z.clone().requires_grad_()
    loss, freq = fn.switch_load_balancing_loss(leaf, topk_indices=idx)
    (dl,) = torch.autograd.grad(loss, leaf)
    _check(loss.detach(), freq, dl, z, ref, torch.float32)
    for bad in (-float("inf"), float("nan"), float("inf")):
        y = z.clone()
        y[5] = bad
        assert torch.isnan(fn.ops.switch_loss(y, topk_indices=idx)[0])


def test_nothing_counts(fn):
    z, idx, _ = _case(50, 24, 3, torch.bfloat16, 1, False)
    none = torch.zeros(50, dtype=torch.bool, device="cuda")
    zero = torch.zeros(24, dtype=torch.int32, device="cuda")
    for kw in (dict(topk_indices=idx, token_mask=none), dict(expert_frequency=zero),
               dict(expert_frequency=zero + 1, token_mask=none)):
        leaf = z.clone().requires_grad_()
        loss, _ = fn.switch_load_balancing_loss(leaf, **kw)
        (dl,) = torch.autograd.grad(loss, leaf)
        assert loss.item() == 0.0 and (dl == 0).all()
    leaf = torch.empty(0, 24, device="cuda", requires_grad=True)
    loss, freq = fn.switch_load_balancing_loss(leaf, topk_indices=idx[:0])
    (dl,) = torch.autograd.grad(loss, leaf)
    assert loss.item() == 0.0 and dl.shape == (0, 24) and (freq == 0).all()


def test_bad_indices_are_reported_and_not_counted(fn):
    z, idx, _ = _case(500, 24, 3, torch.bfloat16, 1, False)
    idx[3, 1], idx[400, 0] = 24, -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    loss, freq, _ = fn.ops.switch_loss(z, topk_indices=idx, err=err)
    ref = obalance.switch_loss(z, idx=idx)
    assert err.item() == 201 and torch.equal(freq.long(), ref[1])
    assert abs(loss.item() - ref[0].item()) <= RTOL * ref[0].item()


def test_unaligned_rows_and_strided_inputs(fn):
    z, idx, _ = _case(400, 64, 4, torch.bfloat16, 9, False)
    ref = fn.ops.switch_loss(z, topk_indices=idx)
    buf = torch.empty(400 * 64 + 3, dtype=torch.bfloat16, device="cuda")
    for off in (1, 2, 3):
        y = buf[off:off + 400 * 64].view(400, 64)
        y.copy_(z)
        got = fn.ops.switch_loss(y, topk_indices=idx)
        assert all(torch.equal(a, b) for a, b in zip(ref, got))
        d = fn.ops.switch_loss_bwd(y, got[2], torch.ones((), device="cuda"))
        assert torch.equal(d, fn.ops.switch_loss_bwd(z, got[2], torch.ones((), device="cuda")))
    wide = torch.zeros(400, 130, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2][:, :64] = z
    leaf = wide[:, ::2][:, :64].detach().requires_grad_()
    loss, freq = fn.switch_load_balancing_loss(leaf, topk_indices=idx.t().contiguous().t().long())
    (dl,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(loss.detach(), ref[0]) and torch.equal(freq, ref[1]) and dl.shape == z.shape


def test_gradient_against_differences(fn):
    """Central differences of the float64 loss, whose own error is O(h^2): the kernel's gradient matches
    them in a random direction."""
    z, idx, mask = _case(90, 20, 3, torch.float32, 11, True)
    leaf = z.clone().requires_grad_()
    loss, _ = fn.switch_load_balancing_loss(leaf, topk_indices=idx, token_mask=mask)
    (dl,) = torch.autograd.grad(loss, leaf)
    g = torch.Generator().manual_seed(0)
    for _ in range(4):
        d = torch.randn(z.shape, generator=g, dtype=torch.float64).cuda()
        h = 1e-5
        up, down = (obalance.switch_loss(z.double() + s * h * d, idx=idx, mask=mask)[0] for s in (1, -1))
        want = ((up - down) / (2 * h)).item()
        got = (dl.double() * d).sum().item()
        scale = (dl.double() * d).abs().sum().item()
        assert abs(got - want) <= 1e-4 * scale


def test_second_derivative(fn):
    """create_graph: the gradient of a function of the gradient, against float64 autograd."""
    z, idx, mask = _case(30, 12, 2, torch.float32, 2, True)
    leaf = z.clone().requires_grad_()
    loss, freq = fn.switch_load_balancing_loss(leaf, topk_indices=idx, token_mask=mask)
    (dl,) = torch.autograd.grad(loss, leaf, create_graph=True)
    (got,) = torch.autograd.grad(dl.square().sum(), leaf)
    ref = z.double().requires_grad_()
    p = torch.softmax(ref, 1) * mask[:, None]
    rl = 12 * (p.sum(0) / p.sum() * (freq.double() / freq.sum())).sum()
    (rdl,) = torch.autograd.grad(rl, ref, create_graph=True)
    (want,) = torch.autograd.grad(rdl.square().sum(), ref)
    assert (got.double() - want).norm() <= 1e-4 * want.norm()


def test_second_derivative_of_left_out_rows(fn):
    """Infinities and NaN in rows that do not count reach neither gradient."""
    z, idx, mask = _case(30, 12, 2, torch.float32, 2, True)
    assert not mask.all()
    second = []
    for fill in (None, float("nan"), float("inf")):
        leaf = z.clone()
        if fill is not None:
            leaf[~mask] = fill
        leaf.requires_grad_()
        loss, _ = fn.switch_load_balancing_loss(leaf, topk_indices=idx, token_mask=mask)
        (dl,) = torch.autograd.grad(loss, leaf, create_graph=True)
        (got,) = torch.autograd.grad(dl.square().sum(), leaf)
        assert (dl[~mask] == 0).all() and (got[~mask] == 0).all()
        second.append(got)
    assert torch.equal(second[0], second[1]) and torch.equal(second[0], second[2])


def test_graph_replays_and_streams(fn):
    """Two captured graphs with their own tensors, replayed in turn on other inputs, and two streams at
    once: the results are the eager ones."""
    cases = [_case(700, 96, 4, torch.bfloat16, s, True) for s in (1, 2)]
    other = [_case(700, 96, 4, torch.bfloat16, s, True) for s in (3, 4)]

    def step(z, idx, mask):
        loss, freq, coef = fn.ops.switch_loss(z, topk_indices=idx, token_mask=mask)
        return loss, freq, fn.ops.switch_loss_bwd(z, coef, torch.ones((), device="cuda"), mask)

    graphs = []
    for c in cases:
        step(*c)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*c)
        graphs.append((g, out))
    for c, o in zip(cases, other):
        for a, b in zip(c, o):
            a.copy_(b)
    want = [step(*o) for o in other]
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for (_, got), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    streams = [torch.cuda.Stream() for _ in other]
    got = []
    for s, o in zip(streams, other):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(*o))
    torch.cuda.synchronize()
    for a, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, w))


def test_module_and_compiled_training_step(fn):
    """The module's auxiliary loss and its router gradient, and the traced loss with its backward."""
    import sonicmoe

    torch.manual_seed(3)
    m = sonicmoe.MoE(8, 2, 512, 256, sonicmoe.ActivationType.SWIGLU, False, 0.02).to(torch.bfloat16).cuda()
    x = torch.randn(200, 512, dtype=torch.bfloat16, device="cuda")
    _, aux = m(x)
    aux.backward()
    logits = torch.nn.functional.linear(x, m.router.weight.detach())
    _, idx = sonicmoe.ops.router_topk(logits, 2)
    rloss, _, rdl, _ = obalance.switch_loss(logits, idx=idx)
    assert abs(aux.item() - rloss.item()) <= RTOL * rloss.item()
    want = rdl.T @ x.double()
    # dlogits and the weight gradient are each rounded to bf16: 2^-8 of the value at most, twice
    assert (m.router.weight.grad.double() - want).norm() <= 2 * 2.0 ** -8 * want.norm()

    def loss_of(z):
        return fn.switch_load_balancing_loss(z, topk_indices=idx)[0]

    leaf = logits.clone().requires_grad_()
    (eager,) = torch.autograd.grad(loss_of(leaf), leaf)
    leaf2 = logits.clone().requires_grad_()
    (compiled,) = torch.autograd.grad(torch.compile(loss_of, fullgraph=True)(leaf2), leaf2)
    assert torch.equal(eager, compiled)
