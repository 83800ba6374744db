"""The polynomial tanh of capped attention scores (tanh_poly2 in attention_packed.cuh), restated in numpy float32 with
the coefficients read from the source: its absolute error on |u| <= 1 stays under 4e-7, so a cap of 50 moves a score by
at most 2e-5."""
import os
import re

import numpy as np

SRC = os.path.join(os.path.dirname(__file__), "..", "ltx-rust_b200", "csrc", "attention_packed.cuh")


def test_tanh_poly():
    text = open(SRC).read()
    c = [np.float32(float.fromhex(v)) for v in re.findall(r"t[0-5] = (-?0x1\.[0-9a-f]+p[-+]\d+)f", text)]
    assert len(c) == 6, "tanh_poly2 coefficients not found"
    u = np.linspace(-1, 1, 400001).astype(np.float32)
    z = (u * u).astype(np.float32)
    q = np.full_like(u, c[5])
    for k in c[4::-1]:
        q = (q * z + k).astype(np.float32)
    got = (q * u).astype(np.float32).astype(np.float64)
    assert np.abs(got - np.tanh(u.astype(np.float64))).max() < 4e-7
