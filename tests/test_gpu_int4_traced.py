"""GPU tests of the functional entry points on 4-bit expert weights traced as a whole graph: the eager results."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [5, 70])
@pytest.mark.parametrize("concat", [False, True])
def test_whole_graphs(T, concat):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import functional as fn

    E, H, I, K = 32, 256, 64, 4
    g = torch.Generator(device="cuda").manual_seed(T)
    w1 = torch.randn(2 * I, H, E, generator=g, device="cuda", dtype=torch.bfloat16) * 0.05
    w2 = torch.randn(H, I, E, generator=g, device="cuda", dtype=torch.bfloat16) * 0.05
    p1, p2 = fn.prepare_int4_weights(w1, 32, concat_glu=concat), fn.prepare_int4_weights(w2, 64)
    rw = torch.randn(E, H, generator=g, device="cuda", dtype=torch.bfloat16) * 0.05
    x = torch.randn(T, H, generator=g, device="cuda", dtype=torch.bfloat16)
    tok = torch.arange(T, device="cuda").repeat_interleave(2)
    ex = torch.randint(0, E, (2 * T,), generator=g, device="cuda")
    sc = torch.rand(2 * T, generator=g, device="cuda")
    kw = dict(is_inference_mode_enabled=True, concat_layout=concat)

    def layer(x):
        return fn.moe_TC_softmax_topk_layer(x, rw, p1, None, p2, None, K, None, **kw)

    def fused(x):
        return fn.moe_TC_softmax_topk_layer(x, rw, p1, None, p2, None, K, None, fused_router=True, **kw)

    def lists(x):
        return fn.moe_general_routing_inputs(x, sc, tok, ex, p1, None, p2, None, E, None, **kw)

    for call in (layer, fused, lists):
        torch._dynamo.reset()
        want, got = call(x), torch.compile(call, fullgraph=True)(x)
        assert len(want) == len(got)
        for a, b in zip(want, got):
            assert a.dtype == b.dtype and torch.equal(a, b)
