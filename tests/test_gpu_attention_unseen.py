"""Attention on a B200: keys that a row does not see, beside infinities that it
does see and beside rows that a call does not compute."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import attention_oracle as ref  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
INF, NAN = math.inf, float("nan")


@pytest.fixture(scope="module")
def at():
    from pspml import attention
    return attention


def _rand(seed, *shape, dtype, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * size).to(dtype)


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device="cuda")


def _cache(at, keys, values, page):
    """The sequences' keys and values in pages of a pool whose other slots hold NaN."""
    need = [(k.shape[0] + page - 1) // page for k in keys]
    _, hkv, dim = keys[0].shape
    pool = torch.full((2, sum(need) + 1, page, hkv, dim), NAN, dtype=keys[0].dtype, device="cuda")
    table = torch.full((len(keys), max(need)), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    first = 1
    for s, (k, v) in enumerate(zip(keys, values)):
        n = k.shape[0]
        j = torch.arange(n, device="cuda")
        table[s, :need[s]] = torch.arange(first, first + need[s], device="cuda")
        pool[0][first + j // page, j % page] = k
        pool[1][first + j // page, j % page] = v
        first += need[s]
    lengths = torch.tensor([k.shape[0] for k in keys], dtype=torch.int32, device="cuda")
    return at.KvCache(pool[0], pool[1]), lengths, table


def _same(out, lse, want, scale8=None, zero8=0):
    """The formula's value: its infinities by sign, NaN where it is NaN, else to the usual
    tolerance; an S8 output clamps infinities and holds the zero point for NaN."""
    o, l, tol_o, tol_l = want
    fine = torch.isfinite(o)
    got = out.double()
    if scale8 is None:
        assert torch.equal(got.isposinf(), o.isposinf()), "+inf"
        assert torch.equal(got.isneginf(), o.isneginf()), "-inf"
        assert torch.equal(got.isnan(), o.isnan()), "NaN"
        over = (got[fine] - o[fine]).abs() - tol_o[fine]
    else:
        assert (got[o.isposinf()] == 127).all(), "+inf"
        assert (got[o.isneginf()] == -128).all(), "-inf"
        assert (got[o.isnan()] == zero8).all(), "NaN"
        exact = (o[fine] / scale8 + zero8).clamp(-128, 127)
        over = (got[fine] - exact).abs() - (0.5 + tol_o[fine] / scale8 + 1e-3)
    assert (over <= 0).all()
    assert torch.isfinite(l).all()
    assert ((lse.double() - l).abs() <= tol_l).all()


# Values of v at tokens from the sequence's begin (>= 0) and end (< 0) in a
# column: rows between see the first ones only.
MIXES = [
    [(0, 5, INF), (-2, 5, NAN)], [(1, 5, -INF), (-3, 5, INF)],
    [(0, 7, INF), (-1, 7, -INF), (-2, 1, NAN)],
    [(0, 2, INF), (1, 2, -INF), (-2, 2, NAN)],        # seen infinities of both signs: NaN
    [(0, None, INF), (-2, None, INF), (-3, 4, NAN)],  # an overflowed token in every column
    [(0, 3, INF), (2, 3, NAN), (-2, 3, INF)]]


def _mix(v, mix):
    for token, column, value in mix:
        v[token, :, slice(None) if column is None else column] = value


def _wants(q, k, v, first, rows, window=0):
    parts = [ref.attend(q[r:r + 1], k, v, first + r, True, window, q.shape[-1] ** -0.5) for r in rows]
    return tuple(torch.cat(x) for x in zip(*parts))


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("tokens,hq,hkv,dim,dtype", [
    (40, 4, 2, 128, BF16), (300, 8, 1, 64, F16), (257, 3, 3, 80, BF16)])
def test_prompt_seen_infinities(ctx, at, mix, tokens, hq, hkv, dim, dtype):
    # Small queries: no weight is small enough to round to 0, which times an infinity is NaN.
    q = _rand(1, tokens, hq, dim, dtype=dtype, size=0.1)
    k, v = _rand(2, tokens, hkv, dim, dtype=dtype), _rand(3, tokens, hkv, dim, dtype=dtype)
    _mix(v, mix)
    out, lse = torch.zeros_like(q), torch.zeros((tokens, hq), device="cuda")
    out8 = torch.zeros((tokens, hq, dim), dtype=torch.int8, device="cuda")
    at.prompt(ctx, q, k, v, _starts([tokens]), out, lse=lse)
    at.prompt(ctx, q, k, v, _starts([tokens]), at.Quantised(out8, 0.02, -3))
    ctx.check_device()
    rows = sorted(set(range(min(8, tokens))) | set(range(max(0, tokens - 140), tokens)))
    want = _wants(q, k, v, 0, rows)
    _same(out[rows], lse[rows], want)
    _same(out8[rows], lse[rows], want, 0.02, -3)


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("bound", [4, 80])  # 80: the tensor-core kernel
@pytest.mark.parametrize("lengths,new,hq,hkv,dim,page,dtype", [
    ([900, 70], [4, 4], 8, 4, 128, 16, BF16), ([90, 300], [4, 3], 4, 1, 64, 8, F16),
    ([20000], [4], 4, 1, 128, 16, BF16)])  # the last: cut over the device
def test_cached_seen_infinities(ctx, at, mix, bound, lengths, new, hq, hkv, dim, page, dtype):
    keys = [_rand(4 + s, n, hkv, dim, dtype=dtype) for s, n in enumerate(lengths)]
    values = [_rand(8 + s, n, hkv, dim, dtype=dtype) for s, n in enumerate(lengths)]
    for v in values:
        _mix(v, mix)
    cache, n, table = _cache(at, keys, values, page)
    q = _rand(12, sum(new), hq, dim, dtype=dtype, size=0.1)
    out, lse = torch.zeros_like(q), torch.zeros((sum(new), hq), device="cuda")
    at.cached(ctx, q, cache, _starts(new), n, table, out, bound, lse=lse)
    ctx.check_device()
    a, parts = 0, []
    for s, m in enumerate(new):
        parts.append(_wants(q[a:a + m], keys[s], values[s], lengths[s] - m, range(m)))
        a += m
    _same(out, lse, tuple(torch.cat(x) for x in zip(*parts)))


@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("computed", [1, 2, 40])  # rows of each sequence that the call computes
@pytest.mark.parametrize("lengths,new,hq,hkv,dim,dtype", [
    ([130, 700, 3], [3, 60, 3], 8, 2, 128, BF16), ([50], [50], 4, 1, 64, F16),
    ([64, 2000, 1], [64, 45, 1], 4, 2, 80, BF16)])
def test_rows_past_max_new_hold_nan(ctx, at, window, computed, lengths, new, hq, hkv, dim, dtype):
    # Keys of the rows that are not computed hold NaN and infinities; those rows stay as they are.
    keys = [_rand(20 + s, n, hkv, dim, dtype=dtype) for s, n in enumerate(lengths)]
    values = [_rand(24 + s, n, hkv, dim, dtype=dtype) for s, n in enumerate(lengths)]
    done = [min(m, computed) for m in new]
    for k, v, n, m, d in zip(keys, values, lengths, new, done):
        if d < m:
            v[n - m + d:] = NAN
            v[n - 1] = INF
            k[n - m + d:, :, 1] = NAN
    cache, n, table = _cache(at, keys, values, 16)
    q = _rand(28, sum(new), hq, dim, dtype=dtype)
    out, lse = torch.full_like(q, 7.0), torch.full((sum(new), hq), 7.0, device="cuda")
    at.cached(ctx, q, cache, _starts(new), n, table, out, computed, lse=lse, window=window)
    ctx.check_device()
    a = 0
    for s, (m, d) in enumerate(zip(new, done)):
        _same(out[a:a + d], lse[a:a + d],
              _wants(q[a:a + d], keys[s], values[s], lengths[s] - m, range(d), window))
        assert (out[a + d:a + m] == 7).all() and (lse[a + d:a + m] == 7).all()
        a += m


@pytest.mark.parametrize("bound", [4, 80])
@pytest.mark.parametrize("lengths,new,hq,hkv,dim,dtype", [
    ([20000], [4], 4, 1, 128, BF16), ([7000, 30], [3, 4], 8, 2, 80, F16)])
def test_cached_not_causal_cut(ctx, at, bound, lengths, new, hq, hkv, dim, dtype):
    # Cut over the device, every row seeing all keys, those of the rows after it too.
    keys = [_rand(40 + s, n, hkv, dim, dtype=dtype) for s, n in enumerate(lengths)]
    values = [_rand(44 + s, n, hkv, dim, dtype=dtype) for s, n in enumerate(lengths)]
    cache, n, table = _cache(at, keys, values, 16)
    q = _rand(48, sum(new), hq, dim, dtype=dtype)
    out, lse = torch.zeros_like(q), torch.zeros((sum(new), hq), device="cuda")
    at.cached(ctx, q, cache, _starts(new), n, table, out, bound, lse=lse, causal=False)
    ctx.check_device()
    a, parts = 0, []
    for s, m in enumerate(new):
        parts.append(ref.attend(q[a:a + m], keys[s], values[s], lengths[s] - m, False, 0, dim ** -0.5))
        a += m
    _same(out, lse, tuple(torch.cat(x) for x in zip(*parts)))


@pytest.mark.parametrize("tokens,hq,hkv,dim,dtype", [(700, 8, 2, 128, BF16), (2600, 1, 1, 64, F16)])
def test_rows_done_again_stay(ctx, at, tokens, hq, hkv, dim, dtype):
    # Other lanes of the warp write a row done again than wrote it first: every time the second
    # writing is the one that stays.  2600 tokens of one head are cut over the device.
    q, k, v = (_rand(32 + i, tokens, h, dim, dtype=dtype) for i, h in enumerate((hq, hkv, hkv)))
    v[::50, :, 1] = NAN
    v[:100] = v[:100].nan_to_num()
    out, lse = torch.zeros_like(q), torch.zeros((tokens, hq), device="cuda")
    at.prompt(ctx, q, k, v, _starts([tokens]), out, lse=lse)
    rows = list(range(0, tokens, 13))
    _same(out[rows], lse[rows], _wants(q, k, v, 0, rows))
    again = torch.empty_like(out)
    for _ in range(30):
        at.prompt(ctx, q, k, v, _starts([tokens]), again.fill_(7))
        assert torch.equal(again.isnan(), out.isnan())
        assert torch.equal(again.nan_to_num(), out.nan_to_num())


def test_rows_done_again_outlast_the_wait_limit(ctx, at):
    # One bad value after a million keys: its tile's rows are done again for longer than the 4 s
    # that any wait in the kernel may take, while other items wait in the same CTA.
    keys, seqs, new, dim, page = 1000040, 300, 20, 8, 512
    need = (keys + page - 1) // page
    g = torch.Generator(device="cuda").manual_seed(30)
    pool = torch.randn((2, need + 1, page, 1, dim), generator=g, device="cuda").to(F16)
    # The sequences share their pages but for the last one of the first sequence.
    table = torch.arange(need, dtype=torch.int32, device="cuda")[None].repeat(seqs, 1)
    pool[:, need] = pool[:, need - 1]
    table[0, -1] = need
    pool[1, need, (keys - 2) % page, 0, 3] = NAN
    q = _rand(31, seqs * new, 1, dim, dtype=F16, size=0.1)
    out, lse = torch.zeros_like(q), torch.zeros((seqs * new, 1), device="cuda")
    lengths = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
    at.cached(ctx, q, at.KvCache(pool[0], pool[1]), _starts([new] * seqs), lengths, table, out, new,
              lse=lse)
    ctx.check_device()
    for s in (0, 1, 147, 148, 149, 150, 151, 298, 299):
        k, v = (pool[i][table[s].long()].view(-1, 1, dim)[:keys] for i in range(2))
        rows = slice(s * new, (s + 1) * new)
        _same(out[rows], lse[rows], _wants(q[rows], k, v, keys - new, range(new)))
    assert torch.isfinite(out[new:]).all()
