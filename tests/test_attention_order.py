"""How the calls of one context are ordered on the device: the library's own
host code on a fake CUDA runtime that logs launches, events and waits."""
import ctypes
import subprocess
from pathlib import Path

import pytest

from pspml import capi

ROOT = Path(__file__).resolve().parents[1]
MAKE = ROOT / "psp-ml_b200"


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    capi.load()  # the built library: its objects are next to it
    names = [x for x in (MAKE / "Makefile").read_text().replace("\\\n", " ").splitlines()
             if x.startswith("SRCS")][0].split(":=")[1].split()
    objects = [MAKE / "_build" / n.replace(".cu", ".o") for n in names]
    if not all(o.exists() for o in objects):
        subprocess.run(["make", "-C", str(MAKE), "-j8"], check=True)
    so = tmp_path_factory.mktemp("fake") / "libpspml_fake.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-I/usr/local/cuda/include", "-o", str(so),
                    str(ROOT / "tests" / "fake_cudart.cpp"), *map(str, objects), "-Wl,-Bsymbolic"],
                   check=True)
    lib = ctypes.CDLL(str(so))
    for name, (res, args) in capi._PROTOS.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    lib.fake_log.restype = ctypes.c_char_p
    return lib


@pytest.fixture
def context(fake):
    ctx = ctypes.c_void_p()
    assert fake.pspml_ctx_create(0, 1 << 20, ctypes.byref(ctx)) == capi.OK
    fake.fake_clear()
    yield ctx
    fake.pspml_ctx_destroy(ctx)


def _cached(fake, ctx, stream, max_new=1):
    """A call that may be split over the device; its pointers are never read on the host."""
    q = capi.Heads(4096, 512, 64, 8, 64, capi.DTYPE_F16, 0, 1.0, 0)
    out = capi.Heads(1 << 20, 512, 64, 8, 64, capi.DTYPE_F16, 0, 1.0, 0)
    cache = capi.KvCacheView(1 << 21, 1 << 22, 2048, 128, 64, 100, 16, 2, 64, capi.DTYPE_F16)
    d = capi.AttentionDesc(0.125, 1, 0, 0)
    assert fake.pspml_attention_cached(
        ctx, ctypes.byref(d), 4, 2, max_new, 4096, 4096, 4096, 100, ctypes.byref(q),
        ctypes.byref(cache), ctypes.byref(out), None, stream) == capi.OK


def _log(fake):
    """(what, stream) of each logged call, a kernel by the part of its name that says which."""
    out = []
    for line in fake.fake_log().decode().splitlines():
        what, stream = line.rsplit(" ", 1)
        for kernel in ("k_attn_step", "k_attn_tc", "k_wait_selftest"):
            if kernel in what:
                what = kernel
        out.append((what, int(stream)))
    return out


@pytest.mark.parametrize("max_new,kernel", [(1, "k_attn_step"), (40, "k_attn_tc")])
@pytest.mark.parametrize("streams", [(7, 9), (2, 2), (7, 7)])
def test_calls_wait_for_the_last_one(fake, context, streams, max_new, kernel):
    # Equal handles need not be one stream: 2 is each host thread's own default stream, and a
    # destroyed stream's handle may come back while its work still runs.
    for s in streams:
        _cached(fake, context, s, max_new)
    a, b = streams
    assert _log(fake) == [(kernel, a), ("record", a), ("wait", b), (kernel, b), ("record", b)]


def test_counters_are_cleared_when_nothing_runs(fake, context):
    # A call made after a kernel gave up may still run on a stream that the clearing does not wait
    # for, and counts on the counters.
    assert fake.pspml_ctx_wait_selftest(context, 1, 0) == capi.OK
    _cached(fake, context, 7)
    fake.fake_clear()
    assert fake.pspml_ctx_check_device(context) == capi.ERR_DEVICE_WAIT
    whats = [what for what, _ in _log(fake)]
    assert "memset" in whats
    assert "synchronize device" in whats[:whats.index("memset")]
    assert fake.pspml_ctx_check_device(context) == capi.OK
