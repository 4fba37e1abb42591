"""The angles of rotations, which torch computes on any device."""
import math

import pytest
import torch

import praghip


def test_rotary_table():
    """The angles in 64 bits; interpolation by parts keeps the fast pairs and divides the slow ones."""
    cos, sin = praghip.rotary_table(1000, 64, theta=1e4, device="cpu")
    for p, i in ((0, 0), (1, 0), (999, 31), (500, 7)):
        angle = p * 1e4 ** (-i / 32)
        assert abs(float(cos[p, i]) - math.cos(angle)) <= 2.0 ** -24 and abs(float(sin[p, i]) - math.sin(angle)) <= 2.0 ** -24
    linear = praghip.rotary_table(1000, 64, theta=1e4, factor=4.0, device="cpu")
    assert float((linear[0][4 * torch.arange(250)] - cos[:250]).abs().max()) <= 2.0 ** -23
    parts = praghip.rotary_table(1000, 64, theta=1e4, factor=4.0, original=4096, device="cpu", magnitude=2.0)
    # pair 0 turns 652 times within 4096 tokens, pair 31 0.09 times
    assert float((parts[0][:, 0] - 2 * cos[:, 0]).abs().max()) <= 2.0 ** -22
    assert float((parts[1][:, 31] - 2 * linear[1][:, 31]).abs().max()) <= 2.0 ** -22
    turns = [4096 * 1e4 ** (-i / 32) / (2 * math.pi) for i in range(32)]
    for i in range(32):
        share = math.acos(float(parts[0][1, i]) / 2) / 1e4 ** (-i / 32) if i < 20 else None
        if share is not None:
            assert 0.2499 <= share <= 1.0001 and (turns[i] < 32 or share > 0.99)
    assert praghip.rotary_table(0, 64, device="cpu")[0].shape == (0, 32) and praghip.rotary_table(5, 0, device="cpu")[0].shape == (5, 0)
    for bad in (dict(theta=0.0), dict(factor=0.0), dict(original=-1), dict(original=100, slow=40.0), dict(original=100, theta=1.0)):
        with pytest.raises(praghip.PraghipError, match="E_ROTARY_SHAPE"):
            praghip.rotary_table(10, 64, device="cpu", **bad)
    with pytest.raises(praghip.PraghipError, match="E_ROTARY_SHAPE"):
        praghip.rotary_table(10, 63, device="cpu")
