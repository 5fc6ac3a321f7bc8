"""The quotient of the 8-bit cache's quantiser (kv8_append.cu, encode8): x r + (x - (x r) s) r with r the float32 nearest
to 1 / s equals the IEEE float32 quotient x / s for every bf16 significand of x and of the block's maximum (the scale is
the maximum times the float32 nearest to 1 / 127 or 1 / 448), over the exponents between them that a code can tell from
zero and beyond.  The fused multiply-adds are restated in wider arithmetic, rounded once: the product q s has 48 bits, so
x - q s is exact in float64; q + rem r needs the 64 bits of extended precision (rem r is below 2^-22 of q, 48 bits)."""
import numpy as np
import pytest


def _fma_remainder(q, s, x):
    return (x.astype(np.float64) - q.astype(np.float64) * s.astype(np.float64)).astype(np.float32)


def _round_sum(q, rem, r):
    exact = q.astype(np.longdouble) + rem.astype(np.longdouble) * r.astype(np.longdouble)
    return exact.astype(np.float32)


@pytest.mark.parametrize("qmax", [127.0, 448.0])
def test_corrected_quotient_is_the_ieee_quotient(qmax):
    sig = np.arange(128, 256, dtype=np.float32)
    top = sig / np.float32(128)  # the block's maximum, up to a power of two (which scales everything exactly)
    s = (top * np.float32(1.0 / qmax)).astype(np.float32)
    r = (np.float32(1) / s).astype(np.float32)
    for e in range(-24, 1):
        x = (sig / np.float32(128) * np.float32(2.0 ** e)).astype(np.float32)
        xx, ss, rr = np.broadcast_arrays(x[None, :], s[:, None], r[:, None])
        q0 = (xx * rr).astype(np.float32)
        q = _round_sum(q0, _fma_remainder(q0, ss, xx), rr)
        assert np.array_equal(q, (xx / ss).astype(np.float32)), e
