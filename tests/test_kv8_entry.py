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


def test_an_empty_batch_is_nothing_to_do():
    """Its tensors have no memory, so their addresses are null."""
    gone = dict(table=0, lens=0, kn=0, vn=0, new_lens=0)
    assert _append(**gone) == 0, _lib.lib().mfd_last_error()
    attend = [0, 256, 128, 128, P, P, 2 * 16 * 128, 16 * 128, 128, _lib.MFD_I8, P, P, 4, 16, 0, 4, 4, 0, 0, 0, 0, 0, 0, 0, 0,
              0, 1, 2, 2, 128, 1.0, 0, 256, 128, 128, 0, P, 1 << 40, P, 1 << 20, 0]
    assert _lib.packed("mfd_kv8_attention", 1)(*attend) == 0, _lib.lib().mfd_last_error()
    weigh = [0, 256, 128, 128, 0, P, 2 * 16 * 128, 16 * 128, 128, _lib.MFD_E4M3, P, 4, 16, 0, 4, 4, 0, 0, 0, 1, 0, 0, 1, 2, 2,
             128, 1.0, 1.0, 0, 0, 4, P, 1 << 20, P, 0, 0]
    assert _lib.packed("mfd_kv8_page_weights", 2)(*weigh) == 0, _lib.lib().mfd_last_error()
    assert _lib.packed("mfd_kv8_evict", 3)(0, 0, 0, 0, 4, 16, 4, 1, 1, 0, 0, 0, 0, 0, 0) == 0, _lib.lib().mfd_last_error()


def test_null_pointers_of_a_batch_are_refused():
    for name in ("k", "v", "ks", "vs", "table", "lens", "kn", "vn", "new_lens"):
        assert _append(bs=1, **{name: 0}) != 0 and b"null" in _lib.lib().mfd_last_error()
