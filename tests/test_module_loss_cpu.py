"""CPU tests of the module's auxiliary loss as a method: subclasses and callers of it are heard.  Stand-ins take
the place of the layer and of the loss's kernels."""
import pytest
import torch
import torch.nn.functional as F

E, H, T = 4, 16, 6


@pytest.fixture
def moe(monkeypatch):
    import sonicmoe
    from sonicmoe import moe as module

    g = torch.Generator().manual_seed(0)
    logits, freq = torch.randn(T, E, generator=g), torch.tensor([5, 1, 2, 4], dtype=torch.int32)
    monkeypatch.setattr(module, "moe_TC_softmax_topk_layer", lambda x, *_: (x, logits, freq))
    monkeypatch.setattr(module, "switch_load_balancing_loss", lambda z, f: (("kernels", z, f), f))

    def build(cls=sonicmoe.MoE):
        return cls(E, 2, H, 8, sonicmoe.ActivationType.SWIGLU, False, 0.02)

    return sonicmoe.MoE, build, logits, freq


def _formula(probs, freq):
    f = freq.float()
    return E * (F.normalize(probs.sum(0), p=1, dim=0) * F.normalize(f, p=1, dim=0)).sum()


def test_the_modules_own_loss_uses_the_kernels(moe):
    _, build, logits, freq = moe
    _, aux = build()(torch.zeros(T, H))
    assert aux[0] == "kernels" and torch.equal(aux[1], logits) and aux[2] is freq
    assert build()(torch.zeros(T, H), is_inference_mode=True)[1] is None


def test_a_subclass_is_heard(moe):
    MoE, build, logits, freq = moe
    seen = []

    class Z(MoE):
        def _compute_switch_loss(self, logits, probs, expert_frequency):
            seen.append((logits, probs, expert_frequency))
            return super()._compute_switch_loss(logits, probs, expert_frequency) + torch.logsumexp(logits, -1).sum()

    _, aux = build(Z)(torch.zeros(T, H))
    probs = F.softmax(logits, -1)
    assert torch.equal(seen[0][0], logits) and torch.equal(seen[0][1], probs) and seen[0][2] is freq
    assert torch.equal(aux, _formula(probs, freq) + torch.logsumexp(logits, -1).sum())


def test_an_instances_own_loss_is_heard(moe):
    _, build, logits, freq = moe
    m = build()
    m._compute_switch_loss = lambda logits, probs, expert_frequency: probs.max()
    assert m(torch.zeros(T, H))[1] == F.softmax(logits, -1).max()


def test_given_probabilities_are_used(moe):
    _, build, logits, freq = moe
    probs = F.softmax(logits / 2, -1).requires_grad_()
    got = build()._compute_switch_loss(logits.view(2, 3, E), probs.view(2, 3, E), freq)
    assert torch.equal(got, _formula(probs, freq))
    assert torch.autograd.grad(got, probs)[0].abs().sum() > 0
