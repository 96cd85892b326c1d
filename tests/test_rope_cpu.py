"""Rotation tables for long contexts: YaRN's ramp against its definition, pair by pair (no GPU)."""
from __future__ import annotations

import math

import numpy as np
import pytest

from m1moe_b200 import rope_table


@pytest.mark.parametrize("rot,theta,original,factor,fast,slow", [
    (128, 1e4, 131072, 4.0, 32, 1),   # the pair that turns once lies beyond the last one
    (128, 1e4, 1000000, 8.0, 32, 1),
    (64, 5e5, 8192, 16.0, 32, 1),     # both ends inside
    (128, 1e4, 100, 4.0, 32, 1),      # no pair turns 32 times
    (64, 1e4, 5, 4.0, 32, 1),         # no pair turns even once
    (128, 1e4, 4096, 2.0, 40, 2),
    (32, 100.0, 32, 4.0, 32, 1),
])
def test_yarn_ramp(rot, theta, original, factor, fast, slow):
    """Pair i turns n theta^(-2i/rot) / 2 pi times in n positions.  Between the pair numbers at which that
    is `fast` and `slow`, in whole pairs, its angle goes linearly from its own to a factor-th of it; the
    others are at one end.  One position's angle is below 1, so the table's sine gives it to 2^-22."""
    t = rope_table(2, rot, theta=theta, device="cpu", scaling={"type": "yarn", "factor": factor, "original": original,
                                                               "beta_fast": fast, "beta_slow": slow}).double()
    gain = 0.1 * math.log(factor) + 1
    pair = np.arange(rot // 2)
    own = theta ** (-2.0 * pair / rot)
    number = lambda turns: rot / 2 * math.log(original / (2 * math.pi * turns)) / math.log(theta)
    first, last = math.floor(number(fast)), math.ceil(number(slow))
    part = np.clip((pair - first) / (last - first), 0.0, 1.0)
    want = own * (1 - part) + own / factor * part
    got = np.arctan2(t[1, :, 1].numpy(), t[1, :, 0].numpy())
    assert np.allclose(got, want, rtol=0, atol=2.0 ** -22)
    assert np.allclose(t[0, :, 0], gain, rtol=1e-6)


def test_yarn_keeps_the_docstrings_promise():
    """Pairs that turn more than beta_fast times stay; those below beta_slow are divided by the factor,
    and none that turns more often than that."""
    t = rope_table(2, 128, theta=1e4, device="cpu", scaling={"type": "yarn", "factor": 4, "original": 131072}).double()
    got = np.arctan2(t[1, :, 1].numpy(), t[1, :, 0].numpy())
    own = 1e4 ** (-np.arange(64) / 64.0)
    turns = 131072 * own / (2 * math.pi)
    assert turns.min() > 2  # every pair turns more than once: none is divided all the way
    assert np.all(got > 0.4 * own)
    assert np.allclose(got[turns > 40], own[turns > 40], rtol=1e-4)
