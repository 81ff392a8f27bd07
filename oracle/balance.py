"""Switch balance loss, per-expert counts and gradient in float64 (the formula of reference
sonicmoe/moe.py:263-276, with an optional token mask)."""
import torch


def switch_loss(logits, freq=None, idx=None, mask=None, dloss=1.0):
    """(loss, counts int64 [E], dlogits, bound) in float64.  ``bound``: dloss * p * max |c|, the size an
    error of c or of its mean has in dlogits."""
    z = logits.detach().double()
    T, E = z.shape
    keep = torch.ones(T, dtype=torch.bool, device=z.device) if mask is None else mask.bool()
    if freq is None:
        ids = idx.long()[keep].reshape(-1)
        ids = ids[(ids >= 0) & (ids < E)]
        freq = torch.bincount(ids, minlength=E)
    freq = freq.long()
    p = torch.zeros_like(z)
    p[keep] = torch.softmax(z[keep], 1)
    n, F = int(keep.sum()), int(freq.sum())
    if n == 0 or F == 0:
        return torch.zeros((), dtype=torch.float64), freq, torch.zeros_like(z), torch.zeros_like(z)
    f = freq.double() / F
    loss = E * (p.sum(0) / n * f).sum()
    c = E * f / n
    dlogits = dloss * p * (c - (p * c).sum(1, keepdim=True))
    return loss, freq, dlogits, abs(dloss) * p * (E * f - 1).abs().max() / n
