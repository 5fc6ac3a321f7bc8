"""The corrected quotient of the quantiser (kv8_append.cu, encode8) for scales that no bf16 maximum gave: within the scales
that it is used for it is the IEEE float32 quotient, outside it need not be.  The fused multiply-adds are libm's fmaf, which
rounds once.  (All 2^23 significands of s against all of x at one power of two were gone through once in C: none differs; other powers
of two scale every step exactly as long as r and the remainder are normal.)"""
import ctypes
import ctypes.util
import random
import re
import os

import numpy as np
import pytest

fmaf = ctypes.CDLL(ctypes.util.find_library("m")).fmaf
fmaf.restype, fmaf.argtypes = ctypes.c_float, [ctypes.c_float] * 3
SOURCE = os.path.join(os.path.dirname(__file__), "..", "mfd_b200", "csrc", "kv8_append.cu")


def _corrected(x, s, r):
    q = float(np.float32(x) * np.float32(r))
    return fmaf(fmaf(q, -s, x), r, q)


def _limits():
    lo, hi = re.search(r"kFastScaleLo = ([0-9.e+-]+)f.*kFastScaleHi = ([0-9.e+-]+)f", open(SOURCE).read()).groups()
    return float(np.float32(lo)), float(np.float32(hi))


@pytest.mark.parametrize("end", ["low", "one", "high"])
def test_the_corrected_quotient_is_the_ieee_quotient_for_every_scale_it_is_used_for(end):
    rng = random.Random(5)
    significands = [0, 1, 2, 3, (1 << 23) - 1, (1 << 23) - 2, (1 << 22), (1 << 22) - 1] + [rng.randrange(1 << 23) for _ in range(60)]
    lo, hi = _limits()
    for m in significands:
        base = np.float32(1 + m * 2.0 ** -23)
        s = {"low": base * np.float32(lo), "one": base, "high": base * np.float32(hi / 2)}[end]
        r = np.float32(1) / s
        assert lo <= s <= hi and r >= np.float32(2.0 ** -126)
        for e in (-11, -10, -1, 0, 1, 6, 8):
            for g in range(128, 256):
                x = g / 128 * 2.0 ** e * float(s / base)
                if x > 3.3e38:
                    continue
                x = np.float32(x)
                assert _corrected(float(x), float(s), float(r)) == float(x / s), (m, e, g)


def test_a_scale_near_the_floor_for_which_it_is_not():
    s = np.float32((2 - 2.0 ** -23) * 2.0 ** -100)
    x = np.float32(2.0 ** -109)
    assert s < _limits()[0] and _corrected(float(x), float(s), float(np.float32(1) / s)) != float(x / s)
