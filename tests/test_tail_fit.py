"""The polynomial of the normal tail that GELU's passes share (csrc/ckpt8.cuh), on the CPU: its constants read
from the source, against erfc in 64 bits."""
import math
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TEXT = open(os.path.join(ROOT, "audiocraft.cpp_b200", "csrc", "ckpt8.cuh")).read()


def constants():
    body = TEXT[TEXT.index("void normal_tail("):]
    body = body[:body.index("q = mul2(r, e);")]
    first = re.search(r"r = pair\((-?[\d.e+-]+)f\);", body).group(1)
    rest = re.findall(r"r = fma2\(r, t, pair\((-?[\d.e+-]+)f\)\);", body)
    c = [np.float32(v) for v in [first] + rest]
    assert len(c) == 9  # degree 8
    return c


Z = np.concatenate([np.linspace(0, 2, 40001), np.linspace(2, 14.5, 50001)])
WANT = np.array([math.exp(z * z / 2) * 0.5 * math.erfc(z / math.sqrt(2)) for z in Z])


def test_fit_is_as_close_as_its_comment_says():
    stated = float(re.search(r"relative error\s+(?://\s*)?([\d.e-]+) for \|z\| <= 14.5", TEXT).group(1))
    t = 1 / (1 + 0.3 * Z)
    p = np.zeros_like(t)
    for c in constants():
        p = p * t + float(c)
    # exp and erfc in 64 bits lose up to z^2 / 2 * 2^-53 and a few steps: 2e-14
    worst = np.abs(p / WANT - 1).max()
    assert worst <= stated + 2e-14 and worst >= 0.95 * stated


@pytest.mark.parametrize("steps", [-1, 0, 1])
def test_evaluation_in_fp32_is_as_close_as_its_comment_says(steps):
    # one rounding per multiply-add; the reciprocal exact or one step off either way
    stated = float(re.search(r"evaluated in fp32 ([\d.e-]+)", TEXT).group(1))
    z = Z.astype(np.float32)
    want = np.array([math.exp(float(v) ** 2 / 2) * 0.5 * math.erfc(float(v) / math.sqrt(2)) for v in z])
    d = (1.0 + z.astype(np.float64) * float(np.float32(0.3))).astype(np.float32)
    t = (1 / d.astype(np.float64)).astype(np.float32)
    if steps:
        t = np.nextafter(t, np.float32(2 if steps > 0 else 0))
    r = np.full_like(t, constants()[0])
    for c in constants()[1:]:
        r = (r.astype(np.float64) * t.astype(np.float64) + float(c)).astype(np.float32)
    assert np.abs(r.astype(np.float64) / want - 1).max() <= stated
