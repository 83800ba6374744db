"""The polynomial tanh of capped attention scores (tanh_poly2, tanh_small2 in attention_packed.cuh), restated in numpy
float32 with the coefficients read from the source: the absolute error stays under 4e-7, so a cap of 50 moves a score
by at most 2e-5."""
import os
import re

import numpy as np

SRC = os.path.join(os.path.dirname(__file__), "..", "ltx-rust_b200", "csrc", "attention_packed.cuh")


def worst(letter, count, limit):
    """The largest error of u q(u^2) on |u| <= limit in float32, for the coefficients named letter0, letter1, ..."""
    c = [np.float32(float.fromhex(v)) for v in re.findall(letter + r"[0-5] = (-?0x1\.[0-9a-f]+p[-+]\d+)f", open(SRC).read())]
    assert len(c) == count, f"coefficients {letter} not found"
    u = np.linspace(-limit, limit, 400001).astype(np.float32)
    z = (u * u).astype(np.float32)
    q = np.full_like(u, c[-1])
    for k in c[-2::-1]:
        q = (q * z + k).astype(np.float32)
    got = (q * u).astype(np.float32).astype(np.float64)
    return np.abs(got - np.tanh(u.astype(np.float64))).max()


def test_tanh_poly():
    assert worst("t", 6, 1.0) < 4e-7


def test_tanh_of_small_scores():
    assert worst("h", 4, 0.5) < 2e-7
