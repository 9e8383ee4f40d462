"""Index and log-sum-exp arrays that are not aligned to their elements would
fault in the kernels: refused on the host.  On a fake CUDA runtime."""
import ctypes

import pytest

from pspml import capi
from test_attention_order import context, fake  # noqa: F401

ref = ctypes.byref


def _view(heads, data=4096, dtype=capi.DTYPE_F16):
    return capi.Heads(data, heads * 64, 64, heads, 64, dtype, 0, 1.0, 0)


CACHE = capi.KvCacheView(1 << 21, 1 << 22, 2048, 128, 64, 100, 16, 2, 64, capi.DTYPE_F16)


def _launched(fake):  # noqa: F811
    return b"launch" in fake.fake_log()


@pytest.mark.parametrize("name", [None, "starts", "lse"])
def test_prompt(fake, context, name):  # noqa: F811
    at = dict(starts=4096, lse=8192)
    if name:
        at[name] += 2
    d = capi.AttentionDesc(0.125, 1, 0, 0)
    status = fake.pspml_attention_prompt(context, ref(d), 4, 1, at["starts"], ref(_view(8)),
                                         ref(_view(2)), ref(_view(2)), ref(_view(8, 1 << 20)),
                                         at["lse"], 7)
    assert status == (capi.ERR_INVALID_ARG if name else capi.OK)
    assert _launched(fake) == (name is None)
    assert not name or name.encode() in fake.pspml_last_error()


@pytest.mark.parametrize("name", [None, "starts", "lengths", "pages", "lse"])
def test_cached(fake, context, name):  # noqa: F811
    at = dict(starts=4096, lengths=4096, pages=4096, lse=8192)
    if name:
        at[name] += 1
    d = capi.AttentionDesc(0.125, 1, 0, 0)
    status = fake.pspml_attention_cached(context, ref(d), 4, 1, 1, at["starts"], at["lengths"],
                                         at["pages"], 8, ref(_view(8)), ref(CACHE),
                                         ref(_view(8, 1 << 20)), at["lse"], 7)
    assert status == (capi.ERR_INVALID_ARG if name else capi.OK)
    assert _launched(fake) == (name is None)
    assert not name or name.encode() in fake.pspml_last_error()


@pytest.mark.parametrize("name", [None, "positions", "slots"])
def test_rotary(fake, context, name):  # noqa: F811
    d = capi.RotaryDesc(64, 64, 0, 0, 10000.0, 1.0, 1.0, 4.0, 0.0, 1.0)
    r = ctypes.c_void_p()
    assert fake.pspml_rotary_create(context, ref(d), ref(r)) == capi.OK
    at = dict(positions=4096, slots=8192)
    if name:
        at[name] += {"positions": 2, "slots": 4}[name]
    want = capi.ERR_INVALID_ARG if name else capi.OK
    q, out = _view(8), _view(8, 1 << 20)
    assert fake.pspml_rotary_append(r, 4, at["positions"], at["slots"], ref(q), ref(out),
                                    ref(_view(2)), ref(_view(2)), ref(CACHE), 7) == want
    if name != "slots":
        assert fake.pspml_rotary_apply(r, 4, at["positions"], ref(q), ref(out), None, None, 7) == want
    assert _launched(fake) == (name is None)
    assert not name or name.encode() in fake.pspml_last_error()
    assert fake.pspml_rotary_destroy(r) == capi.OK
