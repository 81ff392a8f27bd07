"""CPU tests of the module's 4-bit copies: they follow the weights.  Stand-ins take the place of the preparation
(which then keeps the weight's values) and of the layer (which returns what the copies hold)."""
import copy
import gc
import pickle
import weakref

import pytest
import torch
from torch import nn

E, H, I, T = 3, 8, 8, 4


@pytest.fixture
def moe(monkeypatch):
    import sonicmoe
    from sonicmoe import functional as fn
    from sonicmoe.ops import Int4ExpertWeights

    made = []

    def prepare(w, group_size=128, concat_glu=False, out=None):
        made.append(group_size)
        w = w.detach().permute(2, 0, 1).clone()
        if out is not None and out.q.dtype == w.dtype:
            out.q.copy_(w)
            return out
        return Int4ExpertWeights(w, w[:1], tuple(w.shape), group_size, concat_glu)

    def layer(x, logits, w1, w2, K, *_):
        return torch.full_like(x, float(w1.q.double().sum() + 2 * w2.q.double().sum())), torch.zeros(E, dtype=torch.int32)

    monkeypatch.setattr(fn, "prepare_int4_weights", prepare)
    monkeypatch.setattr(fn, "_int4_tc", layer)
    torch.manual_seed(0)
    m = sonicmoe.MoE(E, 2, H, I, sonicmoe.ActivationType.SWIGLU, False, 1.0).to(torch.bfloat16).eval()
    return m, made


def _value(m, call=None):
    with torch.no_grad():
        return (m if call is None else call)(torch.zeros(T, H, dtype=torch.bfloat16), is_inference_mode=True)[0].max().item()


def _want(m):
    v = float(m.c_fc.weight.detach().double().sum() + 2 * m.c_proj.weight.detach().double().sum())
    return torch.tensor(v, dtype=torch.bfloat16).item()


def test_unchanged_weights_are_prepared_once(moe):
    m, made = moe
    assert m.use_int4_experts(64) is m and made == [64, 64]
    for _ in range(3):
        assert _value(m) == _want(m)
    assert made == [64, 64]
    m.use_int4_experts(32)
    assert _value(m) == _want(m) and made == [64, 64, 32, 32]


def _in_place(m):
    with torch.no_grad():
        m.c_fc.weight.mul_(3)


def _other_data(m):
    m.c_proj.weight.data = m.c_proj.weight.data * 5


def _other_parameter(m):
    old, shape = m.c_fc.weight._version, m.c_fc.weight.shape
    del m.c_fc.weight
    gc.collect()
    m.c_fc.weight = nn.Parameter(torch.randn(shape, dtype=torch.bfloat16))
    with torch.no_grad():
        for _ in range(old - m.c_fc.weight._version):  # the same version, perhaps the same address
            m.c_fc.weight.mul_(1)


def _load(m):
    m.load_state_dict({k: v + 1 for k, v in m.state_dict().items()})


def _load_assign(m):
    m.load_state_dict({k: v + 1 for k, v in m.state_dict().items()}, assign=True)


def _type(m):
    m.c_fc.weight.data = m.c_fc.weight.data.float() + 0.25


def _inference(m):
    with torch.inference_mode():
        m.c_fc.weight = nn.Parameter(torch.randn(E, 2 * I, H, dtype=torch.bfloat16), requires_grad=False)


CHANGES = [_in_place, _other_data, _other_parameter, _load, _load_assign, _type, _inference]


@pytest.mark.parametrize("change", CHANGES)
def test_changed_weights_are_prepared_again(moe, change):
    m, made = moe
    m.use_int4_experts(64)
    before, buffers = _value(m), [c.q for c in m._int4_experts.copies]
    change(m)
    assert _value(m) == _want(m) != before
    if change is not _type:  # what a captured graph points to stays
        assert all(a is c.q for a, c in zip(buffers, m._int4_experts.copies))
    n = len(made)
    assert _value(m) == _want(m) and len(made) == n


def test_traced_forward_follows_the_weights(moe):
    m, made = moe
    m.use_int4_experts(64)
    traced = torch.compile(m, fullgraph=True, backend="aot_eager")
    assert _value(m, traced) == _want(m)
    for _ in range(12):  # more often than a graph may be traced again
        _in_place(m)
        assert _value(m, traced) == _want(m)
    _load(m)
    assert _value(m, traced) == _want(m) == _value(m)


@pytest.mark.parametrize("put_away", [
    lambda w: None, lambda w: nn.Parameter(torch.empty(0)), lambda w: nn.Parameter(w.detach().to("meta"))])
def test_weights_put_away_leave_the_copies(moe, put_away):
    m, made = moe
    m.use_int4_experts(64)
    want = _value(m)
    m.c_fc.weight, m.c_proj.weight = put_away(m.c_fc.weight), put_away(m.c_proj.weight)
    assert _value(m) == want and len(made) == 2
    assert _value(m, torch.compile(m, fullgraph=True, backend="aot_eager")) == want
    m2 = pickle.loads(pickle.dumps(copy.deepcopy(m)))
    assert _value(m2) == want and len(made) == 2


def test_weights_emptied_in_place(moe):
    m, made = moe
    m.use_int4_experts(64)
    want = _value(m)
    m.c_fc.weight.data = torch.empty(0)
    assert _value(m) == want
    m.c_fc.weight.data = torch.ones(E, 2 * I, H, dtype=torch.bfloat16)  # back, with other values
    assert _value(m) == _want(m) != want


def test_weights_changed_before_they_were_put_away(moe):
    m, made = moe
    m.use_int4_experts(64)
    _in_place(m)
    m.c_fc.weight.data = torch.empty(0)
    with pytest.raises(RuntimeError, match="put away"):
        _value(m)


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda m: pickle.loads(pickle.dumps(m))])
def test_copies_of_the_module_have_their_own(moe, copied):
    m, made = moe
    m.use_int4_experts(64)
    m2 = copied(m)
    _in_place(m2)
    assert _value(m2) == _want(m2) != _value(m) == _want(m)
    assert m2._int4_experts.handle != m._int4_experts.handle


def test_copies_go_with_the_module(moe):
    from sonicmoe import functional as fn

    m, made = moe
    m.use_int4_experts(64)
    ref, handle = weakref.ref(m._int4_experts), m._int4_experts.handle
    m.use_int4_experts(None)
    gc.collect()
    assert ref() is None and handle not in fn.Int4Copies._known


def test_no_backward_when_traced_either(moe):
    m, made = moe
    m.use_int4_experts(64).train()
    for call in (m, torch.compile(m, backend="aot_eager")):
        with pytest.raises(NotImplementedError):
            call(torch.zeros(T, H, dtype=torch.bfloat16))
