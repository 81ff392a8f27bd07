"""CPU tests of the counts and ids that the balance loss takes: what reaches the kernels, what is refused."""
import pytest
import torch


@pytest.fixture
def seen(monkeypatch):
    """The arguments of ops.switch_loss, which is replaced."""
    from sonicmoe import functional as fn

    calls = []

    def switch_loss(logits, counts=None, idx=None, mask=None, err=None):
        calls.append((counts, idx))
        return torch.zeros(()), torch.zeros(logits.shape[1]) if counts is None else counts.clone(), None

    monkeypatch.setattr(fn.ops, "switch_loss", switch_loss)
    return fn.switch_load_balancing_loss, calls


@pytest.mark.parametrize("given,read", [
    (torch.int32, torch.int32), (torch.int64, torch.int64), (torch.float32, torch.float32),
    (torch.float64, torch.float64), (torch.float16, torch.float32), (torch.bfloat16, torch.float32),
    (torch.int16, torch.int32), (torch.uint8, torch.int32)])
def test_counts_keep_their_values(seen, given, read):
    loss, calls = seen
    f = torch.tensor([0, 1, 3, 100]).to(given)
    if given.is_floating_point:
        f = f / 128
    loss(torch.zeros(2, 4), expert_frequency=f)
    assert calls[0][0].dtype == read and torch.equal(calls[0][0].double(), f.double())


def test_large_counts_do_not_wrap(seen):
    loss, calls = seen
    f = torch.tensor([1 << 40, 1 << 31, 5])
    loss(torch.zeros(2, 3), expert_frequency=f)
    assert torch.equal(calls[0][0], f)


def test_ids_that_int32_cannot_hold_stay_invalid(seen):
    loss, calls = seen
    ids = torch.tensor([[0, 3], [(1 << 32) + 1, -(1 << 32) + 2], [4, -1]])
    loss(torch.zeros(3, 4), topk_indices=ids)
    got = calls[0][1]
    assert got.dtype == torch.int32 and got[0].tolist() == [0, 3]
    assert ((got[1:] < 0) | (got[1:] >= 4)).all()


def test_refusals(seen):
    loss, calls = seen
    z = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="no gradient"):
        loss(z, expert_frequency=torch.ones(3, requires_grad=True))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(ValueError, match="no gradient"):
            loss(z, expert_frequency=dual)
    with pytest.raises(ValueError, match="real numbers"):
        loss(z, expert_frequency=torch.ones(3, dtype=torch.complex64))
    with pytest.raises(ValueError, match="whole numbers"):
        loss(z, topk_indices=torch.zeros(2, 1))
    assert not calls


@pytest.mark.parametrize("T,E,kind,counts,match", [(-1, 8, 0, 16, "T must"), (4, 0, 0, 16, "E must"), (4, 8, 4, 16, "count type"),
                                                   (4, 8, -1, 16, "count type"), (4, 8, 2, None, "null")])
def test_entry_point_refusals(T, E, kind, counts, match):
    import re

    import build  # sonic-moe_b200/build.py

    build.build()
    from sonicmoe import _native as nat

    lib = nat.load()
    rc = lib.sm_switch_loss_counts(16, 0, T, E, None, counts, kind, 16, 16, 16, 1 << 20, None)
    assert rc == nat.SM_EINVAL and re.search(match, lib.sm_last_error().decode())
    rc = lib.sm_switch_loss_counts(16, 0, 5000, 64, None, 16, 2, 16, 16, 256, 100, None)
    assert rc == nat.SM_EINVAL and "workspace too small" in lib.sm_last_error().decode()
