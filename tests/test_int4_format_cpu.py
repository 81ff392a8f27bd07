"""CPU test of what the 4-bit format's short scales cost."""
import torch

from oracle import int4 as oint4


def test_scale_is_at_most_a_sixteenth_wider():
    """Every bf16 maximum of one binade, alone in its group: the scale is amax / 7 rounded up to 5 significant bits,
    so less than 2^-4 above it, and 2% on average (1/32 times the mean of 1/m, ln 2, over even mantissas m)."""
    amax = (1.0 + torch.arange(128, dtype=torch.float64) / 128).repeat_interleave(32).reshape(128, 32)
    _, s = oint4.quantise(amax, 32)
    wider = s[:, 0] * 7 / amax[:, 0] - 1
    assert (wider >= 0).all() and wider.max() < 1 / 16 and wider.max() > 0.055
    assert 0.018 < wider.mean() < 0.025
