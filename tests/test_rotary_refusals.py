"""Rotary descriptors whose numbers pass the range of the types they are
computed in: refused, no device needed."""
import ctypes

import numpy as np
import pytest

from pspml import capi

attention = pytest.importorskip("pspml.attention")


@pytest.mark.parametrize("change,word", [
    (dict(base=5e-324), b"not finite"),                              # base^(-126/128)
    (dict(scaling=1, factor=1e-320), b"not finite"),                 # f / factor
    (dict(scaling=2, base=1e-300, factor=1e-300), b"not finite"),    # base * factor^(128/126) is 0
    (dict(scaling=3, factor=1e-320, original_len=100.0, low=1.0, high=400.0), b"not finite"),
    (dict(amplitude=1e300), b"amplitude"), (dict(amplitude=-1e39), b"amplitude")])
def test_numbers_past_their_types_are_refused(change, word):
    lib = capi.load()
    d = attention.rotary_desc(128)
    for k, v in change.items():
        setattr(d, k, v)
    out = np.zeros(64, np.uint64)
    assert lib.pspml_rotary_frequencies(ctypes.byref(d), out.ctypes.data) == capi.ERR_INVALID_ARG
    assert word in lib.pspml_last_error()
    assert not out.any()


def test_large_numbers_within_them_are_not():
    lib = capi.load()
    d = attention.rotary_desc(128, base=1e300, scaling="linear", factor=1e-30, amplitude=1e38)
    out = np.zeros(64, np.uint64)
    assert lib.pspml_rotary_frequencies(ctypes.byref(d), out.ctypes.data) == capi.OK
