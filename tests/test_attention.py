"""Rotary frequencies and the attention calls' refusals: no device needed."""
import ctypes
import math

import numpy as np
import pytest
from hypothesis import given, settings, strategies as st

from pspml import capi

attention = pytest.importorskip("pspml.attention")


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def _turns(desc):
    return attention.rotary_frequencies(desc).astype(object)


def _near(bits, turns):
    """A 64-bit fraction holds `turns` (modulo 1) to the double's own 2^-53 relative."""
    want = turns % 1.0
    assert abs(int(bits) / 2.0 ** 64 - want) <= 2.0 ** -50 * max(turns, 1e-300) + 2.0 ** -63


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (6, 3.5)])
def test_frequencies_plain(lib, rot, base):
    bits = _turns(attention.rotary_desc(128, rot, base=base))
    assert len(bits) == rot // 2
    for i, b in enumerate(bits):
        _near(b, base ** (-2.0 * i / rot) / (2 * math.pi))


def test_frequencies_scaled(lib):
    rot, base = 64, 10000.0
    plain = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    for b, f in zip(_turns(attention.rotary_desc(64, base=base, scaling="linear", factor=4.0)), plain):
        _near(b, f / 4 / (2 * math.pi))
    wide = base * 8.0 ** (rot / (rot - 2))
    for i, b in enumerate(_turns(attention.rotary_desc(64, base=base, scaling="base", factor=8.0))):
        _near(b, wide ** (-2.0 * i / rot) / (2 * math.pi))
    mixed = 0
    for b, f in zip(_turns(attention.rotary_desc(64, base=base, scaling="parts", factor=8.0,
                                                 original_len=4096, low=1.0, high=4.0)), plain):
        r = 4096 * f / (2 * math.pi)
        if r >= 4:
            want = f
        elif r <= 1:
            want = f / 8
        else:
            g = (r - 1) / 3
            want, mixed = (1 - g) * f / 8 + g * f, mixed + 1
        _near(b, want / (2 * math.pi))
    assert mixed > 0


@settings(max_examples=50, deadline=None)
@given(rot=st.integers(1, 512).map(lambda x: 2 * x), base=st.floats(1.0, 1e8))
def test_frequencies_any(rot, base):
    bits = _turns(attention.rotary_desc(1024, rot, base=base))
    for i in (0, rot // 4, rot // 2 - 1):
        _near(bits[i], base ** (-2.0 * i / rot) / (2 * math.pi))


@pytest.mark.parametrize("change", [
    dict(head_dim=0), dict(head_dim=1025), dict(rot_dim=3), dict(rot_dim=130), dict(rot_dim=-2),
    dict(layout=2), dict(scaling=4), dict(base=0.0), dict(base=math.inf), dict(base=math.nan),
    dict(amplitude=math.inf), dict(scaling=1, factor=0.0), dict(scaling=2, factor=-1.0),
    dict(scaling=2, rot_dim=2, factor=2.0), dict(scaling=3, factor=2.0, original_len=0.0),
    dict(scaling=3, factor=2.0, original_len=100.0, low=4.0, high=4.0)])
def test_rotary_desc_refused(lib, change):
    d = attention.rotary_desc(128)
    for k, v in change.items():
        setattr(d, k, v)
    out = np.zeros(1024, np.uint64)
    assert lib.pspml_rotary_frequencies(ctypes.byref(d), out.ctypes.data) == capi.ERR_INVALID_ARG
    assert lib.pspml_last_error()
    assert not out.any()


def test_rotary_null_refused(lib):
    d = attention.rotary_desc(128)
    assert lib.pspml_rotary_frequencies(None, None) == capi.ERR_INVALID_ARG
    assert lib.pspml_rotary_frequencies(ctypes.byref(d), None) == capi.ERR_INVALID_ARG
    h = ctypes.c_void_p()
    assert lib.pspml_rotary_create(None, ctypes.byref(d), ctypes.byref(h)) == capi.ERR_INVALID_ARG
    assert lib.pspml_rotary_create(None, ctypes.byref(d), None) == capi.ERR_INVALID_ARG
    assert lib.pspml_rotary_apply(None, 1, 16, None, None, None, None, None) == capi.ERR_INVALID_ARG
    assert lib.pspml_rotary_append(None, 1, 16, 16, None, None, None, None, None,
                                   None) == capi.ERR_INVALID_ARG
    assert lib.pspml_rotary_destroy(None) == capi.OK


def _view(heads=8, dim=64, dtype=capi.DTYPE_F16, **change):
    h = capi.Heads(4096, heads * dim, dim, heads, dim, dtype, 0, 1.0, 0)
    for k, v in change.items():
        setattr(h, k, v)
    return h


def _prompt(lib, d=None, tokens=4, sequences=1, starts=4096, **views):
    """pspml_attention_prompt on views that are never dereferenced (refused first)."""
    d = d or capi.AttentionDesc(0.125, 1, 0, 0)
    v = dict(q=_view(), k=_view(2), v=_view(2), out=_view())
    v.update(views)
    refs = [ctypes.byref(v[n]) if v[n] is not None else None for n in ("q", "k", "v", "out")]
    return lib.pspml_attention_prompt(ctypes.c_void_p(4096), ctypes.byref(d), tokens, sequences,
                                      starts, *refs, None, None)


@pytest.mark.parametrize("views,word", [
    (dict(q=None), b"null"), (dict(out=None), b"null"),
    (dict(q=_view(data=None)), b"null"), (dict(q=_view(data=4097)), b"aligned"),
    (dict(q=_view(dtype=9)), b"dtype"), (dict(q=_view(head_stride=-64)), b"stride"),
    (dict(q=_view(heads=0)), b"heads"), (dict(q=_view(reserved=1)), b"reserved"),
    (dict(q=_view(dtype=capi.DTYPE_S8)), b"S8"),
    (dict(k=_view(3), v=_view(3)), b"shapes"), (dict(v=_view(4)), b"shapes"),
    (dict(k=_view(2, 32)), b"shapes"), (dict(k=_view(2, dtype=capi.DTYPE_BF16)), b"types"),
    (dict(out=_view(7)), b"shapes"), (dict(out=_view(dtype=capi.DTYPE_BF16)), b"dtype"),
    (dict(out=_view(dtype=capi.DTYPE_S8, scale=0.0)), b"scale"),
    (dict(out=_view(dtype=capi.DTYPE_S8, zero_point=128)), b"zero point"),
    (dict(out=_view(head_stride=32)), b"overlap"), (dict(out=_view(token_stride=0)), b"overlap")])
def test_prompt_views_refused(lib, views, word):
    assert _prompt(lib, **views) == capi.ERR_INVALID_ARG
    assert word in lib.pspml_last_error()


def test_prompt_arguments_refused(lib):
    desc = capi.AttentionDesc
    for d in (desc(math.nan, 1, 0, 0), desc(math.inf, 1, 0, 0), desc(1.0, 2, 0, 0),
              desc(1.0, 1, -1, 0), desc(1.0, 0, 4, 0), desc(1.0, 1, 0, 1)):
        assert _prompt(lib, d) == capi.ERR_INVALID_ARG
    assert _prompt(lib, tokens=-1) == capi.ERR_INVALID_ARG
    assert _prompt(lib, tokens=1 << 31) == capi.ERR_INVALID_ARG
    assert _prompt(lib, sequences=-1) == capi.ERR_INVALID_ARG
    assert _prompt(lib, starts=None) == capi.ERR_INVALID_ARG
    big = dict(q=_view(8, 264), k=_view(2, 264), v=_view(2, 264), out=_view(8, 264))
    assert _prompt(lib, **big) == capi.ERR_UNSUPPORTED
    wide = _view(1 << 12)
    assert _prompt(lib, tokens=1 << 20, q=wide, out=wide) == capi.ERR_UNSUPPORTED
    d = desc(1.0, 1, 0, 0)
    assert lib.pspml_attention_prompt(None, ctypes.byref(d), 1, 1, 16, None, None, None, None, None,
                                      None) == capi.ERR_INVALID_ARG


def _cache(heads=2, dim=64, page=16, **change):
    c = capi.KvCacheView(4096, 8192, page * heads * dim, heads * dim, dim, 10, page, heads, dim,
                         capi.DTYPE_F16)
    for k, v in change.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("change,word", [
    (dict(k=None), b"null"), (dict(v=8193), b"aligned"), (dict(dtype=capi.DTYPE_S8), b"dtype"),
    (dict(page_size=0), b"page_size"), (dict(pages=-1), b"pages"), (dict(slot_stride=-1), b"stride"),
    (dict(pages=1 << 31), b"pages"), (dict(heads=3), b"shapes"), (dict(head_dim=32), b"shapes"),
    (dict(dtype=capi.DTYPE_BF16), b"types")])
def test_cached_refused(lib, change, word):
    d = capi.AttentionDesc(0.125, 1, 0, 0)
    q, c = _view(), _cache(**change)
    status = lib.pspml_attention_cached(ctypes.c_void_p(4096), ctypes.byref(d), 4, 1, 4, 4096, 4096,
                                        4096, 8, ctypes.byref(q), ctypes.byref(c),
                                        ctypes.byref(_view()), None, None)
    assert status == capi.ERR_INVALID_ARG
    assert word in lib.pspml_last_error()


def test_cached_arguments_refused(lib):
    d = capi.AttentionDesc(0.125, 1, 0, 0)
    q, c = _view(), _cache()

    def run(max_new=4, lengths=4096, pages=4096, stride=8):
        return lib.pspml_attention_cached(ctypes.c_void_p(4096), ctypes.byref(d), 4, 1, max_new, 4096,
                                          lengths, pages, stride, ctypes.byref(q), ctypes.byref(c),
                                          ctypes.byref(_view()), None, None)

    assert run(max_new=-1) == capi.ERR_INVALID_ARG
    assert run(lengths=None) == capi.ERR_INVALID_ARG
    assert run(pages=None) == capi.ERR_INVALID_ARG
    assert run(stride=-1) == capi.ERR_INVALID_ARG


def test_struct_layouts():
    assert ctypes.sizeof(capi.Heads) == 48
    assert ctypes.sizeof(capi.KvCacheView) == 64
    assert ctypes.sizeof(capi.RotaryDesc) == 64
    assert ctypes.sizeof(capi.AttentionDesc) == 16
    packed = attention._pack_heads(4096, 5, 6, 7, 8, 9, -10, 0.5, 0)
    assert packed == bytes(capi.Heads(4096, 5, 6, 7, 8, 9, -10, 0.5, 0))
