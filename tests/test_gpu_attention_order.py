"""Attention calls of one context from several host threads and streams: they
share the context's workspace and run one after another."""
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF16 = torch.bfloat16
PER_THREAD = 2  # cudaStreamPerThread: one handle, another stream in each host thread


@pytest.fixture(scope="module")
def at():
    from pspml import attention
    return attention


def _call(at, seed, keys, hq, hkv, max_new):
    """One token over `keys` keys: a call that is split over the device, as a function of the
    output and the stream."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = keys // 16 + 1
    pool = torch.randn((2, pages, 16, hkv, 128), generator=g, device="cuda").to(BF16)
    q = torch.randn((1, hq, 128), generator=g, device="cuda").to(BF16)
    cache = at.KvCache(pool[0], pool[1])
    starts, lengths = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [keys]))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]

    def run(ctx, out, stream):
        at.cached(ctx, q, cache, starts, lengths, table, out, max_new, stream=stream)
    return run, q


@pytest.mark.parametrize("max_new", [1, 40])
def test_default_streams_of_two_threads(ctx, at, max_new):
    calls = [_call(at, 3 + i, n, 4, 1, max_new) for i, n in enumerate((60000, 9000))]
    want = []
    for run, q in calls:
        want.append(torch.empty_like(q))
        run(ctx, want[-1], 0)
    outs = [[torch.zeros_like(q) for _ in range(60)] for _, q in calls]
    torch.cuda.synchronize()
    turn, errors = threading.Lock(), []

    def work(i):
        try:
            torch.cuda.set_device(0)
            for o in outs[i]:
                with turn:
                    calls[i][0](ctx, o, PER_THREAD)
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ctx.check_device()
    assert not errors
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
