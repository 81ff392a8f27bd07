"""GPU tests of the 4-bit experts on x of every size, with few tokens and with many: channels far larger than the
others, the largest finite numbers, infinities.  A weight whose code is 0 hides its channel completely.

Tolerances: those of tests/test_gpu_int4.py.  The oracle's bound of the fp32 sums goes by |x| |w|, so a channel on
zero codes adds nothing to it, however large.
"""
import pytest
import torch

from oracle import int4 as oint4

pytestmark = pytest.mark.gpu

H, I, E, K = 1024, 256, 4, 2


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import ops as _ops

    return _ops


def _layer(T, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    w2 = (torch.randn(E, H, I, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx = torch.rand(T, E, generator=g, device="cuda").topk(K, 1).indices.to(torch.int32)
    return w1, w2, x, idx, torch.rand(T, K, generator=g, device="cuda") + 0.1


def _run(ops, w1, w2, x, idx, scores, group):
    out, _ = ops.moe_int4_forward(x, scores, idx, ops.weight_prep_int4(w1, group), ops.weight_prep_int4(w2, group))
    tok = torch.arange(x.shape[0], device="cuda").repeat_interleave(K)
    ref, bound = oint4.experts(x, scores.reshape(-1), tok, idx.reshape(-1), oint4.values(w1, group),
                               oint4.values(w2, group), False)
    return out, ref, bound


def _check(out, ref, bound):
    assert torch.isfinite(out).all()
    d = (out.double() - ref).abs()
    assert (d <= 2.0 ** -8 * ref.abs() + 1.01 * bound + 2.0 ** -133).all(), f"max excess {(d - bound).max():.3g}"


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 8, 9, 70])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 3e38])
def test_large_channels_on_zero_codes(ops, T, group, size):
    w1, w2, x, idx, scores = _layer(T, T + group)
    for c in (7, 500, H - 1):
        w1[:, :, c] = 0
        x[:, c] = size if c != 500 else -size
    _check(*_run(ops, w1, w2, x, idx, scores, group))


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("T", [1, 8, 9])
def test_large_intermediate_channels_on_zero_codes(ops, T, group):
    w1, w2, x, idx, scores = _layer(T, T + group)
    for c, size in ((3, 2.0 ** 10), (200, 2.0 ** 30)):
        w1[:, 2 * c:2 * c + 2] *= size
        w2[:, :, c] = 0
    _check(*_run(ops, w1, w2, x, idx, scores, group))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 8, 9])
def test_products_near_the_largest_number(ops, T, group):
    """x of 2e38 in gates of about 1e36: every sum and every output is finite."""
    w1, w2, x, idx, scores = _layer(T, T + group)
    w1[:, 1::2, 40] = 0  # the ups do not see the channel
    x[:, 40] = 2e38
    out, ref, bound = _run(ops, w1, w2, x, idx, scores, group)
    assert ref.abs().max() > 1e34
    _check(out, ref, bound)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 8, 9, 70])
def test_infinity_of_a_channel_is_an_infinity_of_the_output(ops, T, group):
    """All codes of the channel and of the second product are positive, so no term is 0 * inf or inf - inf."""
    w1, w2, x, idx, scores = _layer(T, T + group)
    w1[:, :, 40] = 0.05
    w2 = (w2.abs() + 0.02).to(torch.bfloat16)
    assert (oint4.quantise(w1, group)[0][..., 40] > 0).all() and (oint4.quantise(w2, group)[0] > 0).all()
    plain, _, _ = _run(ops, w1, w2, x, idx, scores, group)
    x[T // 2, 40] = float("inf")
    out, _, _ = _run(ops, w1, w2, x, idx, scores, group)
    rest = [t for t in range(T) if t != T // 2]
    assert (out[T // 2] == float("inf")).all() and torch.equal(out[rest], plain[rest])
