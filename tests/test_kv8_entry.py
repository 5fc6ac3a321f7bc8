"""Checks of the 8-bit cache's C entry points that come before any CUDA call (no GPU)."""
from mfd_b200 import _lib

P = 1 << 20  # a pointer that is never followed


def _append(**kw):
    """mfd_kv8_append for an empty batch."""
    a = dict(k=P, v=P, sc_p=2 * 16 * 128, sc_h=16 * 128, sc_t=128, code=_lib.MFD_I8, ks=P, vs=P, pages=4, page=16, table=P,
             table_stride=4, width=4, lens=P, kn=P, vn=P, sn_b=0, sn_n=256, sn_h=128, n=2, path=0, path_stride=0, rows=2,
             counts=0, bs=0, hkv=2, d=128, new_lens=2 * P, status=0, stream=0)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.packed("mfd_kv8_append", 0)(*a.values())


def test_append_refuses_a_misaligned_status():
    assert _append() == 0 and _append(status=P) == 0
    assert _append(status=P + 1) != 0
    assert b"status" in _lib.lib().mfd_last_error()
