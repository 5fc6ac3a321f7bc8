"""mfd_kv8_call: the operators of the 8-bit cache with their arguments in one array of words (no GPU: what it refuses, and
that an operator's own refusals come through)."""
import struct

import pytest

from mfd_b200 import _lib

OPS = ["mfd_kv8_append", "mfd_kv8_attention", "mfd_kv8_page_weights", "mfd_kv8_evict"]


def _error():
    return _lib.lib().mfd_last_error().decode()


def test_unknown_operators_and_a_null_array_are_refused():
    call = _lib.lib().mfd_kv8_call
    for op in (-1, 4, 99):
        assert call(op, b"\0" * 8, 1) != 0 and "no operator" in _error()
    assert call(0, None, 0) != 0 and "null" in _error()


@pytest.mark.parametrize("op", range(4))
def test_a_wrong_number_of_words_is_refused(op):
    count = len(_lib._SIGS[OPS[op]][1])
    for n in (0, count - 1, count + 1):
        assert _lib.lib().mfd_kv8_call(op, b"\0" * (8 * (count + 1)), n) != 0
        assert f"{n} words" in _error() and str(count) in _error()


@pytest.mark.parametrize("op", range(4))
def test_refusals_are_those_of_the_operator(op):
    args = [0.0 if a is _lib.c_f32 else 0 for a in _lib._SIGS[OPS[op]][1]]
    rc = getattr(_lib.lib(), OPS[op])(*[None if a is _lib.c_vp else x for a, x in zip(_lib._SIGS[OPS[op]][1], args)])
    direct = _error()
    assert _lib.packed(OPS[op], op)(*args) == rc != 0
    assert _error() == direct and OPS[op] in direct


def test_words_that_are_not_numbers_raise():
    with pytest.raises(struct.error):
        _lib.packed("mfd_kv8_evict", 3)(*([None] * 15))
