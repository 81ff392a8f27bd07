"""GPU test of a module on 4-bit experts whose weights change: its outputs are those of a module that was made from
the new weights, eager, traced and in a graph captured anew."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_module_follows_its_weights():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import sonicmoe

    torch.manual_seed(0)
    m = sonicmoe.MoE(8, 2, 256, 128, sonicmoe.ActivationType.SWIGLU, False, 0.02).to(torch.bfloat16).cuda().eval()
    x = torch.randn(40, 256, dtype=torch.bfloat16, device="cuda")
    m.use_int4_experts(64)
    traced = torch.compile(m, fullgraph=True)

    def outputs(module):
        with torch.no_grad():
            return module(x, is_inference_mode=True)[0]

    seen = []
    for step in range(3):
        fresh = copy.deepcopy(m)
        fresh.use_int4_experts(None).use_int4_experts(64)
        want = outputs(fresh)
        # the traced forward comes first: it has to bring the copies up to date by itself
        assert torch.equal(outputs(traced), want) and torch.equal(outputs(m), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = outputs(m)
        graph.replay()
        assert torch.equal(got, want) and all(not torch.equal(want, s) for s in seen)
        seen.append(want)
        with torch.no_grad():
            if step == 0:
                m.c_fc.weight.mul_(1.5)
            else:
                m.load_state_dict({k: v * 1.25 for k, v in m.state_dict().items()})
    weights = [w.weight.data for w in (m.c_fc, m.c_proj)]
    want = outputs(m)
    m.c_fc.cpu(), m.c_proj.cpu()  # put away
    assert torch.equal(outputs(m), want)
    del weights
