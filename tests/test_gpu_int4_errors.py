"""GPU tests of rejected routing entries in layers whose CTAs take several items each of many column blocks,
where every role of the grouped GEMMs waits for the others: the tokens that are all right get their outputs,
whatever the error word holds and whether or not the caller gives one.

Tolerances: those of tests/test_gpu_int4.py (two roundings to bf16 and the oracle's bound).
"""
import pytest
import torch

from oracle import int4 as oint4

pytestmark = pytest.mark.gpu

E, H, I, K = 16, 4096, 512, 4


@pytest.fixture(scope="module")
def layer():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import ops

    g = torch.Generator(device="cuda").manual_seed(5)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    w2 = (torch.randn(E, H, I, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    return (ops, ops.weight_prep_int4(w1, 64), ops.weight_prep_int4(w2, 64), oint4.values(w1, 64),
            oint4.values(w2, 64))


def _tokens(T):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx = torch.rand(T, E, generator=g, device="cuda").topk(K, 1).indices.to(torch.int32)
    return x, idx, torch.rand(T, K, generator=g, device="cuda") + 0.1, \
        torch.arange(T, device="cuda", dtype=torch.int32).repeat_interleave(K)


def _poison(ops, T):
    """The next workspace and output of this size come from memory that holds NaN."""
    n = ops.nat.load().sm_moe_int4_workspace_bytes(T, T * K, H, I, E)
    both = (torch.full((n,), 255, dtype=torch.uint8, device="cuda"),
            torch.full((T, H), float("nan"), dtype=torch.bfloat16, device="cuda"))
    del both


def _check(out, ref, bound):
    assert torch.isfinite(out).all()
    d = (out.double() - ref).abs()
    assert (d <= 2.0 ** -8 * ref.abs() + 1.01 * bound + 2.0 ** -133).all()


# 300 and 2000 tokens take the one-launch routing plan, 5000 the tiled one
@pytest.mark.parametrize("T", [300, 2000, 5000])
@pytest.mark.parametrize("before", [None, 0, 101, 201])
def test_bad_experts_leave_the_other_tokens_right(layer, T, before):
    ops, p1, p2, v1, v2 = layer
    x, idx, scores, tok = _tokens(T)
    idx[0, 0], idx[T - 1, 1], idx[T // 2] = -1, E, 1 << 30
    err = None if before is None else torch.full((1,), before, dtype=torch.int32, device="cuda")
    _poison(ops, T)
    out, _ = ops.moe_int4_forward(x, scores, idx, p1, p2, err=err)
    ref, bound = oint4.experts(x, scores.reshape(-1), tok, idx.reshape(-1), v1, v2, False)
    _check(out, ref, bound)
    assert (out[T // 2] == 0).all() and (err is None or err.item() == (before or 201))


@pytest.mark.parametrize("T", [300, 2000, 5000])
@pytest.mark.parametrize("before", [None, 0, 204])
def test_bad_tokens_leave_the_other_tokens_right(layer, T, before):
    ops, p1, p2, v1, v2 = layer
    x, idx, scores, tok = _tokens(T)
    tok[0], tok[-1] = -5, T
    err = None if before is None else torch.full((1,), before, dtype=torch.int32, device="cuda")
    _poison(ops, T)
    out, _ = ops.moe_int4_general_forward(x, scores.reshape(-1), tok, idx.reshape(-1), p1, p2, err=err)
    ref, bound = oint4.experts(x, scores.reshape(-1), tok, idx.reshape(-1), v1, v2, False)
    _check(out, ref, bound)
    assert err is None or err.item() == 204


@pytest.mark.parametrize("T", [300, 5000])
def test_an_error_of_an_earlier_call_stops_nothing(layer, T):
    ops, p1, p2, v1, v2 = layer
    x, idx, scores, tok = _tokens(T)
    want, _ = ops.moe_int4_forward(x, scores, idx, p1, p2)
    for code in (101, 201, -1):
        err = torch.full((1,), code, dtype=torch.int32, device="cuda")
        _poison(ops, T)
        out, _ = ops.moe_int4_forward(x, scores, idx, p1, p2, err=err)
        assert torch.equal(out, want) and err.item() == code
