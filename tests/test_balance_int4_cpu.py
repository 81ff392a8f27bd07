"""CPU tests of the balance loss and the 4-bit experts: refusals before any device work, and the oracles
against definitions written another way."""
import pytest
import torch

from oracle import balance as obalance
from oracle import int4 as oint4


@pytest.fixture(scope="module")
def nat():
    import build  # sonic-moe_b200/build.py

    build.build()
    from sonicmoe import _native

    return _native


def _err(nat):
    return nat.load().sm_last_error().decode()


@pytest.mark.parametrize("T,E,dtype,idx,K,freq,match", [
    (-1, 8, 0, None, 0, 16, "T must be"),
    (4, 0, 0, None, 0, 16, "E must be"),
    (4, 4097, 0, None, 0, 16, "E must be"),
    (4, 8, 3, None, 0, 16, "dtype"),
    (4, 8, 0, None, 0, None, "either"),
    (4, 8, 0, 16, 2, 16, "either"),
    (4, 8, 0, 16, 0, None, "either"),
    (4, 8, 0, None, -1, 16, "K >= 0"),
    (4, 8, 0, None, 2, None, "null pointer"),
    (1 << 30, 8, 0, 16, 2, None, "2\\^30"),
    (4, 8, 0, None, 0, 16, "null pointer"),
])
def test_switch_loss_refusals(nat, T, E, dtype, idx, K, freq, match):
    import re

    lib = nat.load()
    rc = lib.sm_switch_loss(None, dtype, T, E, None, idx, K, freq, None, None, None, None, 0, None, None)
    assert rc == nat.SM_EINVAL and re.search(match, _err(nat))


def test_switch_loss_workspace_is_checked(nat):
    lib = nat.load()
    need = lib.sm_switch_loss_workspace(5000, 64)
    assert need > 0
    rc = lib.sm_switch_loss(16, 0, 5000, 64, None, None, 0, 16, 16, 16, None, 256, 100, None, None)
    assert rc == nat.SM_EINVAL and "workspace too small" in _err(nat)
    rc = lib.sm_switch_loss_bwd(None, 0, 4, 8, None, None, None, None, None)
    assert rc == nat.SM_EINVAL and "null pointer" in _err(nat)


@pytest.mark.parametrize("E,N,K,group,concat,code", [
    (0, 16, 64, 32, 0, "SM_EINVAL"), (1, 12, 64, 32, 0, "SM_ENOTSUP"), (1, 16, 60, 32, 0, "SM_ENOTSUP"),
    (1, 16, 64, 48, 0, "SM_ENOTSUP"), (1, 24, 64, 32, 1, "SM_EINVAL"), (1, 16, 64, 32, 0, "SM_EINVAL"),
])
def test_weight_prep_int4_refusals(nat, E, N, K, group, concat, code):
    for f in ("sm_weight_prep_int4", "sm_int4_expand"):
        args = (None, E, N, K, group, concat, None, None, None) if "prep" in f else (None, None, E, N, K, group, concat,
                                                                                    None, None)
        assert getattr(nat.load(), f)(*args) == getattr(nat, code)


@pytest.mark.parametrize("change,code,match", [
    (dict(T=-1), "SM_EINVAL", "T >= 0"), (dict(n=-1), "SM_EINVAL", "entries"), (dict(n=(1 << 30) + 1), "SM_EINVAL", "2.30"),
    (dict(H=100), "SM_ENOTSUP", "multiples of 8"), (dict(I=4), "SM_ENOTSUP", "multiples of 8"),
    (dict(g1=16), "SM_ENOTSUP", "group"), (dict(g2=256), "SM_ENOTSUP", "group"), (dict(n=9), "SM_EINVAL", "T\\*K"),
    (dict(freq=None), "SM_EINVAL", "null"), (dict(x=None), "SM_EINVAL", "null"), (dict(x=24), "SM_EINVAL", "aligned"),
    (dict(ws=100), "SM_EINVAL", "workspace too small"),
])
def test_moe_int4_forward_refusals(nat, change, code, match):
    import re

    a = dict(x=256, T=4, H=128, I=64, E=8, K=2, n=8, g1=32, g2=32, freq=256, ws=1 << 30)
    a.update(change)
    rc = nat.load().sm_moe_int4_forward(a["x"], a["T"], a["H"], a["I"], a["E"], a["K"], a["n"], 256, None, 256, 256, 256,
                                        a["g1"], 256, 256, a["g2"], 256, a["freq"], 256, a["ws"], None, None)
    assert rc == getattr(nat, code) and re.search(match, _err(nat)), _err(nat)


def test_python_refusals():
    from sonicmoe import functional as fn
    from sonicmoe import ops

    z = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA tensor"):
        fn.switch_load_balancing_loss(z, expert_frequency=torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match=r"\[E, N, K\]"):
        ops.weight_prep_int4(torch.zeros(16, 64))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.weight_prep_int4(torch.zeros(1, 16, 64))
    w = ops.Int4ExpertWeights(torch.zeros(1), torch.zeros(1), (1, 16, 64), 32, True)
    w2 = ops.Int4ExpertWeights(torch.zeros(1), torch.zeros(1), (1, 64, 8), 32, False)
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="both"):
        fn.moe_TC_softmax_topk_layer(x, torch.zeros(1, 64), w, None, torch.zeros(64, 8, 1), None, 1, None,
                                     is_inference_mode_enabled=True, concat_layout=True)
    with pytest.raises(ValueError, match="concat_layout"):
        fn.moe_TC_softmax_topk_layer(x, torch.zeros(1, 64), w, None, w2, None, 1, None, is_inference_mode_enabled=True)
    with pytest.raises(NotImplementedError, match="prepared"):
        fn.moe_TC_softmax_topk_layer(x.requires_grad_(), torch.zeros(1, 64), w, None, w2, None, 1, None,
                                     concat_layout=True)
    with pytest.raises(NotImplementedError, match="prepared"):
        fn.moe_general_routing_inputs(x, torch.zeros(2), torch.zeros(2), torch.zeros(2), w, None, w2, None, 1, None,
                                      concat_layout=True)
    with pytest.raises(ValueError, match="topk_scores"):
        ops.moe_int4_forward(x, torch.zeros(2, 2), torch.zeros(2, 1, dtype=torch.int32), w, w2)


def test_int4_oracle_properties():
    """codes in [-7, 7]; 7 scales cover the group, 7 of the next smaller 5-bit number do not; every value is a
    bf16 number; a known tie goes to even."""
    g = torch.Generator().manual_seed(0)
    w = (torch.randn(40, 200, generator=g) * torch.exp(3 * torch.randn(40, 1, generator=g))).to(torch.bfloat16)
    for group in (32, 64, 128):
        q, s = oint4.quantise(w, group)
        assert q.abs().max() <= 7
        amax = torch.nn.functional.pad(w.double().abs(), (0, -200 % group)).unflatten(-1, (-1, group)).amax(-1)
        m, e = torch.frexp(s)
        assert ((m * 32) == torch.round(m * 32)).all() and (7 * s >= amax).all()
        assert (7 * torch.ldexp(m - 1 / 32, e) < amax).all()
        v = oint4.values(w, group)
        assert torch.equal(v.to(torch.bfloat16).double(), v)
        assert ((v - w.double()).abs() <= 0.5 * s.repeat_interleave(group, -1)[..., :200]).all()
    v = oint4.values(torch.tensor([[7.0, 2.5, 3.5, -2.5, -0.5, 0.49]]).to(torch.bfloat16), 32)
    assert v.tolist() == [[7, 2, 4, -2, 0, 0]]


def test_balance_oracle_against_autograd():
    g = torch.Generator().manual_seed(0)
    z = torch.randn(50, 9, generator=g, dtype=torch.float64, requires_grad=True)
    idx = torch.rand(50, 9, generator=g).topk(3, 1).indices
    mask = torch.rand(50, generator=g) < 0.5
    loss, freq, dl, _ = obalance.switch_loss(z, idx=idx, mask=mask, dloss=2.0)
    F = torch.nn.functional
    f = F.one_hot(idx[mask], 9).sum((0, 1)).double()
    p = F.softmax(z, -1)[mask].sum(0)
    ref = 9 * (F.normalize(p, p=1, dim=0) * F.normalize(f, p=1, dim=0)).sum()
    (want,) = torch.autograd.grad(2.0 * ref, z)
    assert torch.equal(freq.double(), f)
    assert abs(loss.item() - ref.item()) < 1e-13 and (dl - want).abs().max() < 1e-15
