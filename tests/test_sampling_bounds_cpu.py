"""The error bound by which the sampling kernel calls a top-p edge certain,
recomputed from the roundings that it has to cover."""
import math
import os
import re

import numpy as np

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "minimal-inference_b200", "csrc")


def _constants():
    src = open(os.path.join(CSRC, "sample.cu")).read()
    body = re.search(r"double mass_error\(double m, int tokens\) \{(.*?)\n\}", src, re.S).group(1)
    per_bit, rest = (float(x) for x in re.findall(r"\d\.\d+e-\d+", body.replace("1e-6", "")))
    return per_bit, rest


def test_mass_error_covers_every_rounding():
    """Of a weight 2^-o: three roundings of o, exp2's 2^-22 (its documented bound),
    and the seven fp32 additions of a vector's eight weights."""
    per_bit, rest = _constants()
    assert per_bit >= 3 * math.log(2) * 2.0 ** -24
    assert rest >= 2.0 ** -22 + 7 * 2.0 ** -24


def test_eight_additions_reach_seven_roundings():
    """A vector whose sum loses nearly half a step at each of its seven additions:
    the additions are no smaller order of the bound."""
    v = np.array([2.0 ** -9] + [0.49 * 2.0 ** -32] * 7)
    s = np.float32(0)
    for x in v.astype(np.float32):
        s = np.float32(s + x)
    lost = v.sum() - float(s)
    assert 6.8 * 2.0 ** -24 * 0.98 < lost / v.sum() <= 7 * 2.0 ** -24


def test_weights_are_exact_to_the_stated_2_to_the_minus_39():
    """The kernel's weight, restated: 2^t from a table of 2^(j/32) and the series of
    2^r to r^4, |r| <= 1/64. Its error is the series' rest, (r ln 2)^5 / 120."""
    t = -np.random.default_rng(0).random(400_000) * 40
    k = np.rint(t * 32)
    r = t - k / 32
    ln2 = math.log(2)
    q = ((ln2 ** 4 / 24 * r + ln2 ** 3 / 6) * r + ln2 ** 2 / 2) * r + ln2
    j = k.astype(np.int64)
    w = np.ldexp(np.exp2((j & 31) / 32) * (1 + q * r), j >> 5)
    want = np.exp2(t.astype(np.longdouble))
    err = float(np.abs(w / want - 1).max())
    assert err <= 2.0 ** -39
    assert abs(err / ((ln2 / 64) ** 5 / 120) - 1) < 0.05  # (and no better than the series)
