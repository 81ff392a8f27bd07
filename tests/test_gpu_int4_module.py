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


def _module():
    import sonicmoe

    torch.manual_seed(0)
    m = sonicmoe.MoE(8, 2, 256, 128, sonicmoe.ActivationType.SWIGLU, False, 0.02).to(torch.bfloat16).cuda().eval()
    return m.use_int4_experts(64), torch.randn(40, 256, dtype=torch.bfloat16, device="cuda")


def _of_new_module(m, x):
    fresh = copy.deepcopy(m)
    fresh.use_int4_experts(None).use_int4_experts(64)
    with torch.no_grad():
        return fresh(x, is_inference_mode=True)[0]


def _scale(m, by):
    with torch.no_grad():
        m.c_fc.weight.mul_(by)
        m.c_proj.weight.mul_(by)


@torch.no_grad()
def test_captured_graph_reads_the_copies_made_later():
    m, x = _module()
    m(x, is_inference_mode=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = m(x, is_inference_mode=True)
    _scale(m, 1.5)
    want = _of_new_module(m, x)
    assert torch.equal(m(x, is_inference_mode=True)[0], want)  # brings the copies up to date, where they were
    junk = [torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    graph.replay()
    assert torch.equal(got, want)
    _scale(m, 0.5)
    m.use_int4_experts(64)
    graph.replay()
    assert torch.equal(got, _of_new_module(m, x))
    del junk


@torch.no_grad()
def test_capture_that_finds_changed_weights():
    m, x = _module()
    m(x, is_inference_mode=True)
    _scale(m, 1.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = m(x, is_inference_mode=True)
    want = _of_new_module(m, x)
    assert torch.equal(m(x, is_inference_mode=True)[0], want)  # before any replay
    graph.replay()
    assert torch.equal(got, want)
    _scale(m, 0.5)
    graph.replay()  # the preparation is part of this graph
    want = _of_new_module(m, x)
    assert torch.equal(got, want) and torch.equal(m(x, is_inference_mode=True)[0], want)


@torch.no_grad()
def test_copies_made_on_one_stream_are_used_on_another():
    m, x = _module()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(6):
        _scale(m, 1.25)
        torch.cuda.synchronize()
        outs = []
        for s in streams[:: 1 if i % 2 else -1]:
            with torch.cuda.stream(s):
                if not outs:
                    torch.cuda._sleep(2000000)  # the copies are made late
                outs.append(m(x, is_inference_mode=True)[0])
        torch.cuda.synchronize()
        want = _of_new_module(m, x)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_preparation_into_an_earlier_result():
    from sonicmoe import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    a, b = (torch.randn(2, 32, 72, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    for concat in (False, True):
        p, want = ops.weight_prep_int4(a, 64, concat_glu=concat), ops.weight_prep_int4(b, 64, concat_glu=concat)
        q, scales = p.q, p.scales
        assert ops.weight_prep_int4(b, 64, concat_glu=concat, out=p) is p and p.q is q and p.scales is scales
        assert torch.equal(q, want.q) and torch.equal(scales, want.scales)
        for kw in (dict(group_size=32, concat_glu=concat), dict(group_size=64, concat_glu=not concat)):
            with pytest.raises(ValueError, match="out is of"):
                ops.weight_prep_int4(b, out=p, **kw)
        with pytest.raises(ValueError, match="out is of"):
            ops.weight_prep_int4(b[:1], 64, concat_glu=concat, out=p)
