"""Cases of the operators that this package has beside its FP8 layer: the switch balance loss of the
router with the per-expert counts and the gradient, and the expert products with 4-bit weights.

``own`` false: ``run`` computes an operator in its plain form, elementary torch operations in 32 bits.
``own`` true: ``run`` makes the calls of a user's program.  Formulas:

balance   p = softmax(logits) per token, P_e = sum of p over the tokens that count,
          f_e = the entries routed to expert e, loss = E * sum_e (P_e / sum P) (f_e / sum f);
          dlogits[t, e] = dloss * p[t, e] (c_e - sum_j p[t, j] c_j), c_e = E f_e / (sum f * sum P).
experts   out[t] = sum over t's entries (expert e, score s) of s * W2_e (silu(W1_e^gate x_t) * (W1_e^up x_t)),
          the weights being codes in [-7, 7] times the scale of their group of input columns: the
          smallest number of 5 significant bits (at least 2^-126) that is >= the group's absolute
          maximum / 7, and code = w / scale rounded to nearest, ties to even.
"""
import functools
import math
import os
import sys

import torch

own = False


# ---------------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # the router's loss for one small step: latency of the calls
        dict(name="balance T64 E128", op="balance", T=64, E=128, K=8, dtype="bf16", counts="given", mask=False),
        # one training step of the headline layer, the layer's own expert counts
        dict(name="balance T32768 E128", op="balance", T=32768, E=128, K=8, dtype="bf16", counts="given", mask=False),
        # a padded batch: counts made from the top-k over the tokens that are no padding; odd sizes, fp32 logits
        dict(name="balance T20011 E60 masked", op="balance", T=20011, E=60, K=6, dtype="f32", counts="topk", mask=True),
        # many experts and a long step
        dict(name="balance T131072 E256", op="balance", T=131072, E=256, K=8, dtype="bf16", counts="topk", mask=False),
        # decoding one sequence with the headline layer's experts
        dict(name="experts T1", op="experts", T=1, H=4096, I=1024, E=128, K=8, group=128, concat=False, form="topk",
             zipf=0.0, drop=0.0),
        # a few sequences, Qwen3-style layer, concatenated w1
        dict(name="experts T4 concat", op="experts", T=4, H=2048, I=768, E=128, K=8, group=64, concat=True,
             form="topk", zipf=0.0, drop=0.0),
        # wide experts in small groups, explicit routing lists
        dict(name="experts T16 wide", op="experts", T=16, H=7168, I=2048, E=64, K=8, group=32, concat=False,
             form="lists", zipf=0.0, drop=0.0),
        # odd sizes, tokens without an entry of some experts
        dict(name="experts T33 odd", op="experts", T=33, H=1000, I=408, E=40, K=5, group=64, concat=True,
             form="lists", zipf=0.0, drop=0.3),
        # a decoding batch with unbalanced experts
        dict(name="experts T64 zipf", op="experts", T=64, H=4096, I=1024, E=128, K=8, group=128, concat=False,
             form="lists", zipf=1.2, drop=0.0),
        # the largest decoding batch
        dict(name="experts T512 zipf", op="experts", T=512, H=4096, I=1024, E=128, K=8, group=128, concat=False,
             form="lists", zipf=1.2, drop=0.0),
        # a piece of a prompt through the same 4-bit weights
        dict(name="experts T2048", op="experts", T=2048, H=2048, I=768, E=128, K=8, group=128, concat=True,
             form="topk", zipf=0.0, drop=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        E = _log_int(rng, 4, 512)
        c = dict(op="balance", T=_log_int(rng, 1, 131072), E=E, K=rng.randint(1, min(8, E)),
                 dtype=rng.choice(["bf16", "f16", "f32"]), counts=rng.choice(["given", "topk"]), mask=False)
        while c["T"] * c["E"] > 131072 * 256:
            c["T"] = max(1, c["T"] // 2)
        if c["dtype"] == "f32":
            c["T"] = max(1, c["T"] // 2)
        if c["dtype"] == "f16":
            c["T"] = min(c["T"], 4096)
        c["mask"] = c["counts"] == "topk" and rng.random() < 0.5
        return c
    while True:
        E = _log_int(rng, 4, 128)
        c = dict(op="experts", T=_log_int(rng, 1, 2048), H=8 * _log_int(rng, 16, 896), I=8 * _log_int(rng, 8, 256),
                 E=E, K=rng.randint(1, min(8, E)), group=rng.choice([32, 64, 128]), concat=rng.random() < 0.5,
                 form=rng.choice(["topk", "lists"]), zipf=rng.choice([0.0, 1.2]), drop=0.0)
        if c["form"] == "lists" and rng.random() < 0.5:
            c["drop"] = 0.3
        # within the largest listed weights, products, and products of every token with every expert
        size = c["H"] * c["I"]
        if (E * size <= 128 * 4096 * 1024 and c["T"] * c["K"] * size <= 2048 * 8 * 2048 * 768
                and c["T"] * E * size <= 2048 * 128 * 2048 * 768):
            return c


# ---------------------------------------------------------------------------------------------
# inputs

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _route(case, g, device):
    """Distinct experts [T, K] of every token, drawn without replacement with weights rank^-zipf."""
    T, E, K = case["T"], case["E"], case["K"]
    weight = -case["zipf"] * torch.log(torch.arange(1, E + 1, dtype=torch.float32, device=device))
    weight = weight[torch.randperm(E, generator=g, device=device)]
    u = torch.rand(T, E, generator=g, device=device).clamp_(1e-7, 1.0 - 1e-7)
    return torch.topk(weight - torch.log(-torch.log(u)), K, dim=1).indices.to(torch.int32)


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = _generator(seed)
    s = {"case": case}
    T, E, K = case["T"], case["E"], case["K"]
    if case["op"] == "balance":
        logits = 1.3 * torch.randn(T, E, generator=g, device="cuda") + 0.4 * torch.randn(E, generator=g, device="cuda")
        s["logits"] = logits.to(_DTYPE[case["dtype"]])
        idx = torch.topk(s["logits"].float(), K, dim=1).indices.to(torch.int32)
        s["idx"] = idx if case["counts"] == "topk" else None
        s["freq"] = None if s["idx"] is not None else torch.bincount(idx.reshape(-1), minlength=E).to(torch.int32)
        s["mask"] = None
        if case["mask"]:
            s["mask"] = torch.rand(T, generator=g, device="cuda") < 0.8
        # the loss's weight in the training loss; with fp16 logits times a loss scale that keeps the gradient in range
        s["dloss"] = (0.01 + 0.01 * torch.rand((), generator=g, device="cuda")) * (65536.0 if case["dtype"] == "f16" else 1.0)
        return s
    H, I = case["H"], case["I"]
    s["x"] = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx = _route(case, g, "cuda")
    scores = torch.randn(T, K, generator=g, device="cuda").softmax(1)
    if case["form"] == "topk":
        s["idx"], s["scores"] = idx, scores
    else:
        keep = torch.rand(T, K, generator=g, device="cuda") >= case["drop"]
        s["token"] = torch.arange(T, dtype=torch.int32, device="cuda")[:, None].expand(T, K)[keep].contiguous()
        s["expert"], s["scores"] = idx[keep].contiguous(), scores[keep].contiguous()
    s["w1"] = torch.randn(E, 2 * I, H, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.02)
    s["w2"] = torch.randn(E, H, I, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.02)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "experts":  # the 4-bit weights, laid out once; the bf16 weights are not kept
        w1, w2 = s.pop("w1"), s.pop("w2")
        if own:
            ops = _package().ops
            s["w1"] = ops.weight_prep_int4(w1, case["group"], concat_glu=case["concat"])
            s["w2"] = ops.weight_prep_int4(w2, case["group"])
        else:
            s["w1"], s["w2"] = _quantise(w1, case["group"]), _quantise(w2, case["group"])
    return s


@functools.lru_cache(None)
def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sonic-moe_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sonicmoe
    import sonicmoe.ops

    return sonicmoe


# ---------------------------------------------------------------------------------------------
# one pass

def run(state):
    case = state["case"]
    if case["op"] == "balance":
        return _balance_own(state) if own else _balance_plain(state)
    return _experts_own(state) if own else _experts_plain(state)


def _balance_own(s):
    logits = s["logits"].detach().requires_grad_()
    loss, freq = _package().functional.switch_load_balancing_loss(logits, expert_frequency=s["freq"],
                                                                  topk_indices=s["idx"], token_mask=s["mask"])
    (dlogits,) = torch.autograd.grad(loss, logits, s["dloss"])
    return {"loss": loss.detach(), "freq": freq, "dlogits": dlogits}


def _experts_own(s):
    pkg, case = _package(), s["case"]
    if case["form"] == "topk":
        out, freq = pkg.ops.moe_int4_forward(s["x"], s["scores"], s["idx"], s["w1"], s["w2"])
    else:
        out, freq = pkg.functional.moe_general_routing_inputs(
            s["x"], s["scores"], s["token"], s["expert"], s["w1"], None, s["w2"], None, case["E"], None,
            is_inference_mode_enabled=True, concat_layout=case["concat"])
    return {"out": out, "freq": freq}


def _balance_plain(s):
    E = s["logits"].shape[1]
    x = s["logits"].float()
    p = torch.exp(x - x.max(1, keepdim=True).values)
    p = p / p.sum(1, keepdim=True)
    freq = s["freq"]
    if freq is None:
        one = torch.ones_like(s["idx"]) if s["mask"] is None else s["mask"][:, None].expand_as(s["idx"]).to(torch.int32)
        freq = torch.zeros(E, dtype=torch.int32, device=x.device)
        freq.index_add_(0, s["idx"].reshape(-1), one.reshape(-1).to(torch.int32))
    if s["mask"] is not None:
        p = p * s["mask"][:, None]
    total = p.sum(0)
    f = freq.float() / freq.float().sum().clamp_min(1e-12)
    norm = total.sum().clamp_min(1e-12)
    loss = E * (total / norm * f).sum()
    c = E * f / norm
    dlogits = s["dloss"] * p * (c - (p * c).sum(1, keepdim=True))
    return {"loss": loss, "freq": freq, "dlogits": dlogits.to(s["logits"].dtype)}


def _quantise(w, group):
    """(codes + 8 two to a byte, even column in the low half; scales) of w [E, N, K], rows padded to whole groups."""
    E, N, K = w.shape
    pad = -K % group
    v = torch.nn.functional.pad(w, (0, pad)).float().view(E, N, -1, group)
    amax = v.abs().amax(-1)
    scale = ((amax / 7.0).view(torch.int32) & ~0x7FFFF).view(torch.float32)  # 5 significant bits, toward zero
    scale = torch.where(7.0 * scale < amax, (scale.view(torch.int32) + 0x80000).view(torch.float32), scale)
    scale = torch.where(amax > 0, scale.clamp_min(2.0 ** -126), 0.0)
    code = torch.where(scale[..., None] > 0, v.div_(scale[..., None]).round_(), 0.0).to(torch.int8)
    code = (code + 8).to(torch.uint8).view(E, N, K + pad)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, K


def _dequantise(packed, experts):
    codes, scale, K = packed
    codes, scale = codes[experts], scale[experts]
    q = torch.stack((codes & 15, codes >> 4), -1).view(*scale.shape, -1).float() - 8.0
    return q.mul_(scale[..., None]).view(codes.shape[0], codes.shape[1], -1)[..., :K]


def _experts_plain(s):
    case, x = s["case"], s["x"].float()
    T, I, E = case["T"], case["I"], case["E"]
    if case["form"] == "topk":
        expert = s["idx"].reshape(-1).long()
        token = torch.arange(T, device=x.device).repeat_interleave(case["K"])
    else:
        expert, token = s["expert"].long(), s["token"].long()
    freq = torch.zeros(E, dtype=torch.int32, device=x.device)
    freq.index_add_(0, expert, torch.ones_like(expert, dtype=torch.int32))
    active, slot = torch.unique(expert, return_inverse=True)
    A = active.numel()
    h = torch.matmul(x, _dequantise(s["w1"], active).transpose(1, 2))[slot, token]  # [entries, 2I]
    gate, up = (h[:, :I], h[:, I:]) if case["concat"] else (h[:, 0::2], h[:, 1::2])
    a = gate / (1.0 + torch.exp(-gate)) * up * s["scores"].reshape(-1, 1)
    dense = torch.zeros(A * T, I, device=x.device).index_add_(0, slot * T + token, a).view(A, T, I)
    w2 = _dequantise(s["w2"], active)  # [A, H, I]
    out = torch.matmul(dense.transpose(0, 1).reshape(T, A * I), w2.transpose(1, 2).reshape(A * I, -1))
    return {"out": out.to(torch.bfloat16), "freq": freq}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "balance":
        z, E = s["logits"].double(), case["E"]
        keep = torch.ones(z.shape[0], dtype=torch.bool, device=z.device) if s["mask"] is None else s["mask"]
        if s["freq"] is None:
            f = torch.stack([((s["idx"] == e) & keep[:, None]).sum() for e in range(E)])
        else:
            f = s["freq"]
        f64, n = f.double() / max(1, int(f.sum())), max(1, int(keep.sum()))
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        p = logp.exp() * keep[:, None]
        loss = E * torch.dot(p.sum(0) / n, f64)
        mean = (p * f64).sum(1, keepdim=True)
        grad = s["dloss"].double() * E / n * p * (f64 - mean)
        return {"loss": loss, "freq": f.to(torch.int32), "dlogits": grad}
    x, T = s["x"].double(), case["T"]
    if case["form"] == "topk":
        expert = s["idx"].reshape(-1)
        token = torch.arange(T * case["K"], device=x.device) // case["K"]
    else:
        expert, token = s["expert"], s["token"].long()
    score = s["scores"].reshape(-1).double()
    out = torch.zeros(T, case["H"], dtype=torch.float64, device=x.device)
    freq = []
    for e in range(case["E"]):
        at = (expert == e).nonzero()[:, 0]
        freq.append(at.numel())
        if not at.numel():
            continue
        h = x[token[at]] @ _values64(s["w1"][e], case["group"]).T
        n = case["I"]
        gate, up = (h[:, :n], h[:, n:]) if case["concat"] else (h[:, ::2], h[:, 1::2])
        a = gate * torch.sigmoid(gate) * up
        out.index_add_(0, token[at], score[at, None] * (a @ _values64(s["w2"][e], case["group"]).T))
    return {"out": out, "freq": torch.tensor(freq, dtype=torch.int32)}


def _values64(w, group):
    """The values that the 4-bit form of w [N, K] stands for."""
    w = w.double()
    parts = []
    for k in range(0, w.shape[1], group):
        v = w[:, k:k + group]
        m, e = torch.frexp(v.abs().amax(1, keepdim=True) / 7.0)  # m in [1/2, 1): 5 bits are multiples of 1/32
        step = torch.ldexp(torch.ceil(m * 32.0) / 32.0, e).clamp_min(2.0 ** -126)
        parts.append(torch.round(v / step) * step)
    return torch.cat(parts, 1)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without

@functools.lru_cache(None)
def _entries(T, E, K, zipf, drop):
    """(experts that a routing of these sizes reaches, its entries), from one fixed draw."""
    g = torch.Generator().manual_seed(1)
    idx = _route(dict(T=T, E=E, K=K, zipf=zipf), g, "cpu")
    idx = idx[torch.rand(T, K, generator=g) >= drop]
    return int(torch.unique(idx).numel()), int(idx.numel())


def work(case):
    T, E, K = case["T"], case["E"], case["K"]
    if case["op"] == "balance":
        size = 4 if case["dtype"] == "f32" else 2
        other = 4 * T * K + 4 * E if case["counts"] == "topk" else 8 * E
        return {"bytes": 2 * T * E * size + other + (T if case["mask"] else 0) + 8, "flops": 12 * T * E}
    H, I = case["H"], case["I"]
    active, entries = _entries(T, E, K, case["zipf"], case["drop"])
    groups = 2 * I * -(-H // case["group"]) + H * -(-I // case["group"])
    weights = active * (3 * H * I // 2 + 2 * groups)
    return {"bytes": weights + 4 * T * H + entries * (8 if case["form"] == "topk" else 12) + 4 * E,
            "flops": entries * 6 * H * I}
