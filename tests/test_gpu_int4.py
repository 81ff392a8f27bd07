"""GPU tests of the 4-bit expert weights: the prepared form bit for bit, the layer against float64 on
the weight values it stands for.

Tolerances of the layer.  The intermediate is rounded to bf16 (2^-8 of each value at most) and the output
once; the products are exact and their sums fp32.  Element by element the output is within 2^-8 of itself
plus the oracle's bound (the absolute sum over the intermediate's roundings).  Over a whole output the two
roundings are independent and at most 2^-8 / sqrt(3) of a value in the root mean square: sqrt(2) * 2^-8 /
sqrt(3) = 3.2e-3 in the Frobenius norm, 4e-3 with room for the spread of small outputs.
"""
import pytest
import torch

from oracle import int4 as oint4

pytestmark = pytest.mark.gpu

REL_FRO = 4e-3


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from sonicmoe import ops as _ops

    return _ops


def _weights(E, H, I, seed, std=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device="cuda") * std).to(torch.bfloat16)
    w2 = (torch.randn(E, H, I, generator=g, device="cuda") * std).to(torch.bfloat16)
    return w1, w2, g


def _routing(T, E, K, g, skew=0.0):
    w = -skew * torch.log(torch.arange(1, E + 1, device="cuda").float())
    u = torch.rand(T, E, generator=g, device="cuda").clamp_(1e-6, 1 - 1e-6)
    idx = (w - torch.log(-torch.log(u))).topk(K, 1).indices.to(torch.int32)
    return idx, torch.rand(T, K, generator=g, device="cuda") + 0.1


def _check(out, ref, bound):
    assert out.dtype == torch.bfloat16
    d = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (d <= 2.0 ** -8 * ref.abs() + 1.01 * bound + 2.0 ** -133).all(), f"max excess {(d - bound).max():.3g}"
    if ref.numel() >= 2000:
        assert d.norm() <= REL_FRO * ref.norm(), f"rel {(d.norm() / ref.norm()).item():.3e}"


@pytest.mark.parametrize("E,N,K", [(1, 16, 128), (2, 24, 8), (3, 40, 136), (2, 256, 1000), (4, 512, 512), (1, 8, 4096)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_prepared_weights_bit_exact(ops, E, N, K, group):
    g = torch.Generator(device="cuda").manual_seed(E + N + K)
    w = (torch.randn(E, N, K, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    w[0, 3] = 0
    w[0, 5, :8] = torch.tensor([3.5, -3.5, 7, 2.5, 1.5, -0.5, 0.5, 4.5], device="cuda")  # scale 1: ties
    w[0, 5, 8:] = 0
    w[-1, 0, :] *= 2.0 ** -120  # tiny
    w[-1, 1, :] *= 2.0 ** 120
    w[-1, 2, 0] = 1e-40  # alone in its group: the smallest scale
    w[-1, 2, 1:] = 0
    for concat in (False, True) if N % 16 == 0 else (False,):
        p = ops.weight_prep_int4(w, group, concat_glu=concat)
        v = ops.int4_expand(p)
        assert p.shape == (E, N, K) and p.group_size == group and p.concat_glu == concat
        assert torch.equal(v.double(), oint4.values(w, group))


def test_non_finite_weights_show(ops):
    w = torch.randn(1, 32, 256, device="cuda").to(torch.bfloat16)
    w[0, 4, 5], w[0, 9, 200] = float("inf"), float("nan")
    v = ops.int4_expand(ops.weight_prep_int4(w, 64))
    bad = torch.zeros(32, 256, dtype=torch.bool, device="cuda")
    bad[4, :64] = True
    bad[9, 192:] = True
    assert torch.equal(torch.isnan(v[0]), bad)


LAYER = [
    # T, H, I, E, K, group, concat, skew
    (1, 128, 64, 4, 2, 32, False, 0.0),
    (1, 4096, 1024, 16, 8, 128, False, 0.0),
    (2, 8, 8, 1, 1, 32, False, 0.0),
    (3, 136, 24, 5, 3, 64, True, 0.0),
    (7, 1000, 408, 6, 2, 32, True, 0.0),
    (8, 512, 256, 3, 3, 64, False, 0.0),
    (9, 512, 256, 3, 2, 128, True, 0.0),
    (17, 2048, 768, 12, 8, 64, True, 0.0),
    (33, 264, 72, 9, 4, 32, False, 1.2),
    (64, 1024, 512, 32, 8, 128, False, 1.2),
    (100, 512, 1032, 4, 2, 128, True, 0.0),
    (300, 640, 128, 16, 6, 64, False, 1.2),
    (1000, 256, 256, 7, 3, 128, False, 1.2),
    (40, 64, 24, 1100, 4, 32, False, 0.0),  # more experts, more entries than the one-launch routing plan takes
    (5000, 64, 16, 9, 7, 64, True, 1.2),
    (10, 64, 24, 4096, 2, 64, False, 0.0),  # the most experts, on both paths
    (3, 64, 24, 4096, 8, 32, False, 0.0),
]


@pytest.mark.parametrize("T,H,I,E,K,group,concat,skew", LAYER)
def test_layer_topk(ops, T, H, I, E, K, group, concat, skew):
    w1, w2, g = _weights(E, H, I, T + H + I)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx, scores = _routing(T, E, K, g, skew)
    p1, p2 = ops.weight_prep_int4(w1, group, concat_glu=concat), ops.weight_prep_int4(w2, group)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, freq = ops.moe_int4_forward(x, scores, idx, p1, p2, err=err)
    tok = torch.arange(T, device="cuda").repeat_interleave(K)
    ref, bound = oint4.experts(x, scores.reshape(-1), tok, idx.reshape(-1), oint4.values(w1, group),
                               oint4.values(w2, group), concat)
    assert err.item() == 0 and torch.equal(freq.long(), torch.bincount(idx.reshape(-1), minlength=E))
    _check(out, ref, bound)
    again, _ = ops.moe_int4_forward(x, scores, idx, p1, p2)
    assert torch.equal(out, again)  # the same bits every time


@pytest.mark.parametrize("T", [6, 7])
def test_few_tokens_of_a_large_layer(ops, T):
    """Either side of the size from which a few tokens on groups of 32 take the path for many."""
    H, I, E, K = 4096, 1024, 64, 8
    w1, w2, g = _weights(E, H, I, T)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx = torch.arange(T * K, device="cuda", dtype=torch.int32).reshape(T, K).contiguous()
    scores = torch.rand(T, K, generator=g, device="cuda") + 0.1
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 32)
    out, _ = ops.moe_int4_forward(x, scores, idx, p1, p2)
    # the tokens' experts are all different: the last token's alone, as a layer of its own
    e = slice((T - 1) * K, T * K)
    ref, bound = oint4.experts(x[-1:], scores[-1], torch.zeros(K, device="cuda"), torch.arange(K, device="cuda"),
                               oint4.values(w1[e], 32), oint4.values(w2[e], 32), False)
    _check(out[-1:], ref, bound)


@pytest.mark.parametrize("T,H,I,E,n", [(1, 128, 64, 4, 1), (1, 256, 64, 3, 9), (5, 72, 40, 3, 4), (40, 512, 256, 8, 133),
                                       (64, 256, 128, 70, 500), (8, 512, 256, 4, 256), (8, 512, 256, 4, 257), (200, 264, 136, 5, 700), (900, 128, 64, 6, 2500)])
def test_layer_lists(ops, T, H, I, E, n):
    """Explicit lists: tokens without entries, tokens with many, the same expert twice for a token."""
    w1, w2, g = _weights(E, H, I, T + n)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    tok = torch.randint(0, T, (n,), generator=g, device="cuda").sort().values.to(torch.int32)
    ex = torch.randint(0, E, (n,), generator=g, device="cuda").to(torch.int32)
    sc = torch.randn(n, generator=g, device="cuda")
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 64)
    out, freq = ops.moe_int4_general_forward(x, sc, tok, ex, p1, p2)
    ref, bound = oint4.experts(x, sc, tok, ex, oint4.values(w1, 32), oint4.values(w2, 64), False)
    assert torch.equal(freq.long(), torch.bincount(ex, minlength=E))
    _check(out, ref, bound)


@pytest.mark.parametrize("T", [4, 60, 400, 8300])
def test_bad_entries_are_reported_and_left_out(ops, T):
    E, H, I, K = 6, 256, 64, 2
    w1, w2, g = _weights(E, H, I, T)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx, scores = _routing(T, E, K, g)
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 32)
    v1, v2 = oint4.values(w1, 32), oint4.values(w2, 32)
    tok = torch.arange(T, device="cuda", dtype=torch.int32).repeat_interleave(K)
    bad = idx.clone()
    bad[0, 0], bad[T - 1, 1], bad[1, 0], bad[1, 1] = -1, E, 1 << 30, -(1 << 31)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, freq = ops.moe_int4_forward(x, scores, bad, p1, p2, err=err)
    ref, bound = oint4.experts(x, scores.reshape(-1), tok, bad.reshape(-1), v1, v2, False)
    _check(out, ref, bound)
    assert err.item() == 201 and (out[1] == 0).all()
    ok = bad.reshape(-1)[(bad.reshape(-1) >= 0) & (bad.reshape(-1) < E)]
    assert torch.equal(freq.long(), torch.bincount(ok, minlength=E))
    t2 = tok.clone()
    t2[0], t2[-1] = -5, T
    err.zero_()
    out, _ = ops.moe_int4_general_forward(x, scores.reshape(-1), t2, idx.reshape(-1), p1, p2, err=err)
    ref, bound = oint4.experts(x, scores.reshape(-1), t2, idx.reshape(-1), v1, v2, False)
    _check(out, ref, bound)
    assert err.item() == 204


@pytest.mark.parametrize("T", [8, 9, 80])
def test_infinite_and_nan_tokens_stay_in_their_rows(ops, T):
    E, H, I, K = 4, 264, 72, 2
    w1, w2, g = _weights(E, H, I, T)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx, scores = _routing(T, E, K, g)
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 32)
    ref, _ = ops.moe_int4_forward(x, scores, idx, p1, p2)
    y = x.clone()
    y[2], y[5, 7] = float("nan"), float("inf")
    out, _ = ops.moe_int4_forward(y, scores, idx, p1, p2)
    rest = [t for t in range(T) if t not in (2, 5)]
    assert torch.equal(out[rest], ref[rest]) and torch.isnan(out[2]).all() and not torch.isfinite(out[5]).all()


def test_empty_inputs(ops):
    E, H, I = 5, 128, 64
    w1, w2, _ = _weights(E, H, I, 1)
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 32)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    x = torch.randn(3, H, device="cuda").to(torch.bfloat16)
    out, freq = ops.moe_int4_general_forward(x, none.float(), none, none, p1, p2)
    assert (out == 0).all() and (freq == 0).all()
    out, freq = ops.moe_int4_forward(x[:0], none.float().view(0, 2), none.view(0, 2), p1, p2)
    assert out.shape == (0, H) and (freq == 0).all()


def test_graph_replays_and_streams(ops):
    """Two captured graphs replayed in turn on changed inputs, and two streams at once."""
    E, H, I, K = 8, 512, 256, 4
    w1, w2, g = _weights(E, H, I, 3)
    p1, p2 = ops.weight_prep_int4(w1, 64), ops.weight_prep_int4(w2, 64)
    for T in (2, 150):
        mk = lambda: (torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16), *_routing(T, E, K, g)[::-1])  # noqa: E731
        cases, other = [mk(), mk()], [mk(), mk()]
        graphs = []
        for c in cases:
            ops.moe_int4_forward(*c, p1, p2)
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                o = ops.moe_int4_forward(*c, p1, p2)
            graphs.append((gr, o))
        for c, o in zip(cases, other):
            for a, b in zip(c, o):
                a.copy_(b)
        want = [ops.moe_int4_forward(*o, p1, p2) for o in other]
        for _ in range(2):
            for gr, _ in graphs:
                gr.replay()
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
        streams, got = [torch.cuda.Stream() for _ in other], []
        for s, o in zip(streams, other):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(ops.moe_int4_forward(*o, p1, p2))
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a[0], w[0]) and torch.equal(a[1], w[1])


def test_outputs_into_given_tensors_leave_the_rest(ops):
    E, H, I, K, T = 4, 256, 64, 2, 5
    w1, w2, g = _weights(E, H, I, 3)
    p1, p2 = ops.weight_prep_int4(w1, 64), ops.weight_prep_int4(w2, 64)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx, scores = _routing(T, E, K, g)
    ref, _ = ops.moe_int4_forward(x, scores, idx, p1, p2)
    buf = torch.full((T + 3, H), 7.0, dtype=torch.bfloat16, device="cuda")
    out, _ = ops.moe_int4_forward(x, scores, idx, p1, p2, out=buf[1:T + 1])
    assert torch.equal(buf[1:T + 1], ref) and (buf[0] == 7).all() and (buf[T + 1:] == 7).all()


@pytest.mark.parametrize("concat", [False, True])
def test_functional_layer_and_lists(ops, concat):
    """The functional entry points on prepared 4-bit weights: the layer equals router + experts, the fused
    router is accepted, general routing lists give the same output."""
    from sonicmoe import functional as fn

    E, H, I, K, T = 32, 512, 128, 4, 21
    w1, w2, g = _weights(E, H, I, 8)
    rw = (torch.randn(E, H, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    p1 = fn.prepare_int4_weights(w1.permute(1, 2, 0), 64, concat_glu=concat)
    p2 = fn.prepare_int4_weights(w2.permute(1, 2, 0), 64)
    o, logits, freq = fn.moe_TC_softmax_topk_layer(x, rw, p1, None, p2, None, K, None, is_inference_mode_enabled=True,
                                                   is_softmax_over_topk=False, norm_topk_probs=True, concat_layout=concat)
    sc, idx = ops.router_topk(logits, K, False, True)
    tok = torch.arange(T, device="cuda").repeat_interleave(K)
    ref, bound = oint4.experts(x, sc.reshape(-1), tok, idx.reshape(-1), oint4.values(w1, 64), oint4.values(w2, 64), concat)
    _check(o, ref, bound)
    assert torch.equal(freq.long(), torch.bincount(idx.reshape(-1), minlength=E))
    o2, f2 = fn.moe_general_routing_inputs(x, sc.reshape(-1), tok, idx.reshape(-1), p1, None, p2, None, E, None,
                                           is_inference_mode_enabled=True, concat_layout=concat)
    assert torch.equal(o, o2) and torch.equal(freq, f2)
    o3, lg3, _ = fn.moe_TC_softmax_topk_layer(x, rw, p1, None, p2, None, K, None, is_inference_mode_enabled=True,
                                              concat_layout=concat, fused_router=True)
    sc, idx = ops.router_topk(lg3, K)
    ref, bound = oint4.experts(x, sc.reshape(-1), tok, idx.reshape(-1), oint4.values(w1, 64), oint4.values(w2, 64), concat)
    _check(o3, ref, bound)


def test_module_runs_both_operators(ops):
    """An evaluated module on 4-bit experts: its output, its balance loss with the layer's own counts and
    the router's gradient of that loss; then back to the FP8 engine."""
    import sonicmoe
    from oracle import balance as obalance

    torch.manual_seed(0)
    E, K, H, I = 8, 2, 512, 256
    m = sonicmoe.MoE(E, K, H, I, sonicmoe.ActivationType.SWIGLU, False, 0.02).to(torch.bfloat16).cuda().eval()
    x = torch.randn(3, 11, H, dtype=torch.bfloat16, device="cuda")
    fp8, _ = m(x, is_inference_mode=True)
    assert m.use_int4_experts(64) is m
    o, aux = m(x)
    flat = x.view(-1, H)
    logits = torch.nn.functional.linear(flat, m.router.weight.detach())
    sc, idx = ops.router_topk(logits, K)
    tok = torch.arange(33, device="cuda").repeat_interleave(K)
    ref, bound = oint4.experts(flat, sc.reshape(-1), tok, idx.reshape(-1), oint4.values(m.c_fc.weight.detach(), 64),
                               oint4.values(m.c_proj.weight.detach(), 64), False)
    _check(o.detach().view(-1, H), ref, bound)
    rloss, _, rdl, _ = obalance.switch_loss(logits, idx=idx)
    assert abs(aux.item() - rloss.item()) <= 2.5e-5 * rloss.item()
    aux.backward()
    want = rdl.T @ flat.double()
    assert (m.router.weight.grad.double() - want).norm() <= 2 * 2.0 ** -8 * want.norm()
    with torch.no_grad():
        compiled, aux_c = torch.compile(m, fullgraph=True)(x)
    assert torch.equal(compiled, o.detach()) and torch.allclose(aux_c, aux.detach())
    with pytest.raises(NotImplementedError):
        m.train()(x)
    m.eval().use_int4_experts(None)
    back, _ = m(x, is_inference_mode=True)
    assert (back - fp8).abs().max() <= 2.0 ** -6 * fp8.abs().max()  # bf16 sums in any order, as before


def test_prepared_buffers_are_checked(ops):
    """Buffers that do not belong to the shape and the group are refused before anything runs."""
    import dataclasses

    w1, w2, g = _weights(2, 128, 64, 0)
    p1, p2 = ops.weight_prep_int4(w1, 32), ops.weight_prep_int4(w2, 32)
    x = torch.randn(3, 128, generator=g, device="cuda").to(torch.bfloat16)
    idx, scores = _routing(3, 2, 1, g)
    for change in (dict(q=p1.q[:-16]), dict(scales=p1.scales[:-8]), dict(group_size=64), dict(group_size=0),
                   dict(scales=p1.scales.cpu()), dict(q=p1.q.cpu()), dict(q=p1.q.to(torch.int32)),
                   dict(scales=p1.scales.float()), dict(shape=(4, 128, 128))):
        bad = dataclasses.replace(p1, **change)
        with pytest.raises(ValueError):
            ops.moe_int4_forward(x, scores, idx, bad, p2)
        with pytest.raises(ValueError):
            ops.int4_expand(bad)
