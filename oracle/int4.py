"""4-bit expert weights with group scales and the layer on them, in float64.

A weight is code * scale: scale is the smallest number of 5 significant bits (at least 2^-126) that is
>= amax / 7 of its group of input columns, code = weight / scale to nearest, ties to even.
"""
import torch


def quantise(w, group):
    """(codes int64 [.., K], scales float64 [.., ceil(K / group)]) of w [.., K]."""
    v = torch.nn.functional.pad(w.double(), (0, -w.shape[-1] % group)).unflatten(-1, (-1, group))
    amax = v.abs().amax(-1)
    m, e = torch.frexp(amax / 7.0)  # m in [1/2, 1): 5 significant bits are the multiples of 1/32
    s = torch.ldexp(torch.ceil(m * 32.0) / 32.0, e).clamp_min(2.0 ** -126)
    s = torch.where(amax > 0, s, torch.zeros_like(s))
    q = torch.where(amax[..., None] > 0, torch.round(v / s[..., None].clamp_min(2.0 ** -126)), 0.0)
    return q.long().flatten(-2)[..., : w.shape[-1]], s


def values(w, group):
    """The numbers the 4-bit form of w stands for."""
    q, s = quantise(w, group)
    return q.double() * s.repeat_interleave(group, -1)[..., : w.shape[-1]]


def experts(x, scores, tokens, experts_, w1, w2, concat):
    """(out [T, H], bound [T, H]) of the layer on weight values w1 [E, 2I, H], w2 [E, H, I] and entries
    (token, expert, score); entries with an expert or a token out of range are left out.

    ``bound``: what rounding each intermediate value to bf16 (2^-8 relative at most) and fp32 sums can
    change, as a sum of absolute values."""
    x = x.double()
    T, H = x.shape
    I = w2.shape[2]
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    acc = 2.0 ** -23 * (H / 8 + 64)
    for e in range(w1.shape[0]):
        at = ((experts_ == e) & (tokens >= 0) & (tokens < T)).nonzero()[:, 0]
        if not at.numel():
            continue
        t, s = tokens[at].long(), scores[at].double()[:, None]
        h, habs = x[t] @ w1[e].T, x[t].abs() @ w1[e].abs().T
        pick = (lambda m: (m[:, :I], m[:, I:])) if concat else (lambda m: (m[:, 0::2], m[:, 1::2]))
        (g, u), (ga, ua) = pick(h), pick(habs)
        sg = torch.sigmoid(g)
        a = g * sg * u
        # |silu'| <= 1.1
        a_err = 2.0 ** -8 * a.abs() + acc * (1.1 * u.abs() * ga + (g * sg).abs() * ua)
        out.index_add_(0, t, s * (a @ w2[e].T))
        bound.index_add_(0, t, s.abs() * ((a_err + 2.0 ** -23 * (I / 8 + 64) * a.abs()) @ w2[e].abs().T))
    return out, bound
