"""The stream that the torch mirror's calls are made on: a library that only
records its arguments, no device."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
from pspml import attention  # noqa: E402


class _Library:
    """Every function returns 0 and leaves its last argument, the stream."""

    def __getattr__(self, name):
        def call(*args):
            self.stream = args[-1]
            return 0
        return call


def _calls(lib):
    """The mirror's four calls on CPU tensors (device -1)."""
    ctx = SimpleNamespace(device=-1, handle=None, lib=lib)
    rotary = SimpleNamespace(ctx=ctx, handle=None)
    x = torch.zeros((3, 2, 8), dtype=torch.float16)
    ints = torch.zeros(3, dtype=torch.int32)
    starts = torch.tensor([0, 3], dtype=torch.int32)
    pool = torch.zeros((2, 4, 2, 8), dtype=torch.float16)
    cache = attention.KvCache(pool, pool.clone())
    return [
        lambda **k: attention.rotary_apply(rotary, ints, x, x, **k),
        lambda **k: attention.rotary_append(rotary, ints, ints.long(), x, x, x, x, cache, **k),
        lambda **k: attention.prompt(ctx, x, x, x, starts, x, **k),
        lambda **k: attention.cached(ctx, x, cache, starts, ints[:1], ints[None], x, 3, **k)]


@pytest.mark.parametrize("which", range(4))
def test_calls_go_to_the_current_stream(monkeypatch, which):
    # The stream that torch makes the tensors on: a side stream does not wait for the legacy one.
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device=None: SimpleNamespace(cuda_stream=77))
    lib = _Library()
    call = _calls(lib)[which]
    call()
    assert lib.stream == 77
    for stream in (0, 5):
        call(stream=stream)
        assert lib.stream == stream
