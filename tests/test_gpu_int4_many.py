"""GPU test of the 4-bit experts with more tokens than one launch of the sum over a token's experts takes."""
import pytest
import torch

from oracle import int4 as oint4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lists", [False, True])
def test_many_tokens(lists):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import ops

    T, H, I, E, K = 70001, 64, 24, 5, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device="cuda") * 0.1).to(torch.bfloat16)
    w2 = (torch.randn(E, H, I, generator=g, device="cuda") * 0.1).to(torch.bfloat16)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx = torch.rand(T, E, generator=g, device="cuda").topk(K, 1).indices.to(torch.int32)
    scores = torch.rand(T, K, generator=g, device="cuda") + 0.1
    tok = torch.arange(T, device="cuda", dtype=torch.int32).repeat_interleave(K)
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 32)
    if lists:
        keep = torch.rand(T * K, generator=g, device="cuda") < 0.7
        tok, ex, sc = tok[keep].contiguous(), idx.reshape(-1)[keep].contiguous(), scores.reshape(-1)[keep].contiguous()
        out, freq = ops.moe_int4_general_forward(x, sc, tok, ex, p1, p2)
    else:
        ex, sc = idx.reshape(-1), scores.reshape(-1)
        out, freq = ops.moe_int4_forward(x, scores, idx, p1, p2)
    ref, bound = oint4.experts(x, sc, tok, ex, oint4.values(w1, 32), oint4.values(w2, 32), False)
    assert torch.equal(freq.long(), torch.bincount(ex, minlength=E))
    assert ((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * bound + 2.0 ** -133).all()
