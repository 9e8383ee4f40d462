"""Rotary positions, the paged cache append and attention on a B200 against
plain 64-bit implementations (attention_oracle), over types, head layouts,
lengths, strides, pages and masks."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import attention_oracle as ref  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


@pytest.fixture(scope="module")
def at():
    from pspml import attention
    return attention


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, dtype=F32, size=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * size).to(dtype)


def _close(got, want, tol, what):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: {(~torch.isfinite(got)).sum()} non-finite"
    over = (got - want).abs() - tol
    worst = over.argmax()
    assert over.max() <= 0, (f"{what}: {(over > 0).sum()} of {over.numel()} off, worst "
                             f"{got.flatten()[worst]} for {want.flatten()[worst]} "
                             f"(allowed {tol.flatten()[worst]})")


def _close_lse(got, want, tol):
    empty = torch.isinf(want)
    assert torch.equal(torch.isinf(got.double()) & (got < 0), empty)
    _close(got[~empty], want[~empty], tol[~empty], "lse") if (~empty).any() else None


# ------------------------------------------------------------------ rotary

def _freq(base, rot, scaling, factor=4.0):
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    return f / factor if scaling == "linear" else f


ROTARY = [
    # tokens, hq, hkv, dim, rot, layout, in, out
    (1, 1, 1, 2, 2, "half", F32, F32), (1, 32, 8, 128, 128, "half", BF16, BF16),
    (7, 5, 1, 128, 64, "interleaved", F16, F16), (33, 4, 2, 80, 80, "half", F16, F16),
    (130, 8, 8, 64, 64, "interleaved", BF16, BF16), (9, 3, 3, 96, 48, "half", BF16, BF16),
    (5, 2, 1, 66, 34, "half", F16, F16), (5, 2, 1, 63, 20, "interleaved", BF16, BF16),
    (17, 4, 4, 256, 256, "half", F16, F16), (300, 28, 4, 128, 128, "half", F32, BF16),
    (4, 2, 2, 64, 0, "half", BF16, BF16), (3, 1, 1, 1, 0, "half", F16, F16),
    (12, 6, 2, 1024, 1024, "half", BF16, BF16), (40, 3, 1, 72, 72, "interleaved", F32, F32),
    (65, 4, 4, 128, 32, "interleaved", BF16, F32)]


@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,layout,tin,tout", ROTARY)
def test_rotary(ctx, at, tokens, hq, hkv, dim, rot, layout, tin, tout):
    g = _gen(1)
    q, k = _rand(g, tokens, hq, dim, dtype=tin), _rand(g, tokens, hkv, dim, dtype=tin)
    pos = torch.randint(0, 1 << 20, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    r = at.Rotary(ctx, dim, rot, layout, base=10000.0, scaling="linear", factor=4.0, amplitude=1.25)
    qo = torch.full((tokens, hq, dim), NAN, device="cuda", dtype=tout)
    ko = torch.full((tokens, hkv, dim), NAN, device="cuda", dtype=tout)
    at.rotary_apply(r, pos, q, qo, k, ko)
    torch.cuda.synchronize()
    f = _freq(10000.0, rot, "linear")
    for x, o in ((q, qo), (k, ko)):
        want = ref.rotate(x, pos, rot, layout, f, 1.25)
        _close(o, want, ref.rotary_tolerance(x, rot, tout, 1.25), "rotary")
        assert torch.equal(o[..., rot:], x[..., rot:].to(tout))  # passed through
    qo2 = torch.full_like(qo, NAN)
    at.rotary_apply(r, pos, q, qo2)
    assert torch.equal(qo, qo2)


def test_rotary_far_and_negative_positions(ctx, at):
    # Angles stay exact at any position: 2^31 - 1 turns the fastest pair 3.4e8 times.
    pos = torch.tensor([0, 1, 2 ** 31 - 1, -1, -2 ** 31, 1234567890], dtype=torch.int32, device="cuda")
    q = _rand(_gen(2), 6, 2, 128)
    out = torch.empty_like(q)
    r = at.Rotary(ctx, 128)
    at.rotary_apply(r, pos, q, out)
    bits = at.rotary_frequencies(r.desc)
    # Reference from the same 64-bit fractions in exact integers: the doubles of an angle at 2^31
    # radians are themselves only good to 5e-7.
    angle = torch.tensor([[((p * int(b)) % (1 << 64)) / 2.0 ** 64 * 2 * math.pi for b in bits]
                          for p in pos.tolist()], dtype=torch.float64, device="cuda")
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    x, y = q.double()[..., :64], q.double()[..., 64:]
    want = torch.cat((x * c - y * s, x * s + y * c), dim=-1)
    _close(out, want, ref.rotary_tolerance(q, 128, F32), "far positions")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides_alignment_in_place(ctx, at, layout):
    g = _gen(3)
    r = at.Rotary(ctx, 64, 32, layout)
    f = _freq(10000.0, 32, "none")
    pos = torch.arange(11, dtype=torch.int32, device="cuda")
    fused = _rand(g, 11, 9, 64, dtype=BF16)          # slices of one projection's output
    buf = _rand(g, 11 * 9 * 64 + 1, dtype=BF16)
    odd = buf[1:].view(11, 9, 64)                    # 2-byte aligned only
    swapped = _rand(g, 9, 11, 64, dtype=BF16).transpose(0, 1)
    wide = _rand(g, 11, 9, 67, dtype=BF16)[..., :64]  # rows 134 bytes apart
    for x in (fused, odd, swapped, wide):
        q, k = x[:, :5], x[:, 5:7]
        want_q, want_k = (ref.rotate(t, pos, 32, layout, f) for t in (q, k))
        tol_q, tol_k = (ref.rotary_tolerance(t, 32, BF16) for t in (q, k))
        untouched = x[:, 7:].clone()
        qo = torch.empty((11, 5, 64), dtype=BF16, device="cuda")
        ko = torch.empty((2, 11, 64), dtype=BF16, device="cuda").transpose(0, 1)
        at.rotary_apply(r, pos, q, qo, k, ko)
        _close(qo, want_q, tol_q, "strided q")
        _close(ko, want_k, tol_k, "strided k")
        at.rotary_apply(r, pos, q, q, k, k)          # in place
        assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(x[:, 7:], untouched)


@pytest.mark.parametrize("order", ["slots", "heads"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,page,tin,tout", [
    (1, 8, 2, 64, 64, 16, F16, F16), (77, 28, 4, 128, 128, 16, "s8", F16),
    (50, 4, 4, 80, 40, 5, BF16, BF16), (200, 6, 2, 128, 128, 64, "s8", BF16),
    (19, 3, 1, 33, 6, 8, F32, F32), (700, 0, 8, 128, 128, 32, BF16, BF16)])
def test_append(ctx, at, order, tokens, hq, hkv, dim, rot, page, tin, tout):
    g = _gen(4)
    pages = tokens // page + 3
    quant = tin == "s8"
    if quant:
        x = torch.randint(-128, 128, (tokens, hq + 2 * hkv, dim), device="cuda", generator=g,
                          dtype=torch.int8)
        value = 0.03125 * (x.float() + 7)            # exact in 32 bits
        give = lambda t: at.Quantised(t, 0.03125, -7)  # noqa: E731
    else:
        x = _rand(g, tokens, hq + 2 * hkv, dim, dtype=tin)
        value = x
        give = lambda t: t  # noqa: E731
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    pos = torch.randint(0, 100000, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens].clone()
    skipped = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    if tokens > 10:                                  # slots outside the cache are skipped
        slots[3], slots[7], slots[9] = -1, pages * page, 2 ** 40
        skipped[[3, 7, 9]] = True
    shape = (pages, page, hkv, dim) if order == "slots" else (pages, hkv, page, dim)
    pools = [torch.full(shape, 99.0, device="cuda", dtype=tout) for _ in range(2)]
    kp, vp = pools if order == "slots" else [p.transpose(1, 2) for p in pools]
    r = at.Rotary(ctx, dim, rot)
    f = _freq(10000.0, rot, "none")
    qo = torch.full((tokens, hq, dim), NAN, device="cuda", dtype=tout) if hq else None
    at.rotary_append(r, pos, slots, give(q) if hq else None, qo, give(k), give(v),
                     at.KvCache(kp, vp))
    torch.cuda.synchronize()
    if hq:
        _close(qo, ref.rotate(value[:, :hq], pos, rot, "half", f),
               ref.rotary_tolerance(value[:, :hq], rot, tout), "q")
    kv, vv = value[:, hq:hq + hkv], value[:, hq + hkv:]
    used = slots[~skipped]
    got = kp[used // page, used % page]
    _close(got, ref.rotate(kv, pos, rot, "half", f)[~skipped],
           ref.rotary_tolerance(kv, rot, tout)[~skipped], "cached k")
    assert torch.equal(vp[used // page, used % page], vv[~skipped].to(tout))
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[used] = False
    for p in (kp, vp):
        assert (p.reshape(pages * page, hkv, dim)[rest] == 99.0).all()


# --------------------------------------------------------------- attention

def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device="cuda")


def _check_out(got, lse, wants, scale8=None, zero8=0):
    want = torch.cat([w[0] for w in wants])
    tol = torch.cat([w[2] for w in wants])
    if scale8 is None:
        _close(got, want, tol, "attention")
    else:
        exact = (want / scale8 + zero8).clamp(-128, 127)
        _close(got, exact, 0.5 + tol / scale8 + 1e-3, "attention S8")
    _close_lse(lse, torch.cat([w[1] for w in wants]), torch.cat([w[3] for w in wants]))


PROMPT = [
    # lengths, hq, hkv, dim, dtype, causal, window
    ([1], 1, 1, 64, F16, True, 0), ([2], 2, 1, 128, BF16, True, 0),
    ([37], 8, 2, 64, F16, True, 0), ([128], 4, 4, 128, BF16, True, 0),
    ([129, 1, 127, 0, 64], 8, 2, 128, BF16, True, 0), ([300, 5], 7, 1, 80, F16, True, 0),
    ([257], 6, 2, 96, BF16, False, 0), ([400], 4, 1, 64, F16, True, 33),
    ([200, 200], 16, 1, 128, BF16, True, 1), ([513], 5, 5, 128, F16, True, 256),
    ([64, 65], 3, 1, 8, F16, True, 0), ([90], 2, 2, 112, BF16, True, 40),
    ([70, 3], 4, 2, 192, BF16, True, 0), ([50], 2, 1, 256, F16, True, 7),
    ([45, 60], 3, 3, 33, F16, True, 0), ([66], 4, 2, 64, F32, True, 0),
    ([31, 40], 2, 1, 20, F32, False, 0), ([19], 160, 1, 64, BF16, True, 0),
    ([600], 12, 4, 72, F16, True, 500), ([1000, 24], 8, 1, 128, BF16, False, 0)]


@pytest.mark.parametrize("lengths,hq,hkv,dim,dtype,causal,window", PROMPT)
def test_prompt(ctx, at, lengths, hq, hkv, dim, dtype, causal, window):
    g = _gen(5)
    t = sum(lengths)
    x = _rand(g, t, hq + 2 * hkv, dim, dtype=dtype, size=1.5)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    starts = _starts(lengths)
    out = torch.full((t, hq, dim), NAN, device="cuda", dtype=dtype)
    lse = torch.full((t, hq), NAN, device="cuda")
    at.prompt(ctx, q, k, v, starts, out, lse=lse, causal=causal, window=window)
    torch.cuda.synchronize()
    ctx.check_device()
    wants, a = [], 0
    for n in lengths:
        wants.append(ref.attend(q[a:a + n], k[a:a + n], v[a:a + n], 0, causal, window, dim ** -0.5))
        a += n
    _check_out(out, lse, wants)
    again = torch.full_like(out, NAN)
    at.prompt(ctx, q, k, v, starts, again, causal=causal, window=window)
    assert torch.equal(out, again)                    # same bits from call to call


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (192, BF16)])
def test_prompt_s8_output(ctx, at, dim, dtype):
    g = _gen(6)
    q, k, v = (_rand(g, 150, h, dim, dtype=dtype, size=2.0) for h in (6, 2, 2))
    out = torch.full((150, 6, dim), 55, device="cuda", dtype=torch.int8)
    lse = torch.empty((150, 6), device="cuda")
    at.prompt(ctx, q, k, v, _starts([100, 50]), at.Quantised(out, 0.02, -5), lse=lse)
    wants = [ref.attend(q[a:b], k[a:b], v[a:b], 0, True, 0, dim ** -0.5)
             for a, b in ((0, 100), (100, 150))]
    _check_out(out, lse, wants, 0.02, -5)
    assert (out == 127).any() and (out == -128).any()  # clamped at both ends


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_neighbours_hold_nan(ctx, at, dim):
    # A sequence full of NaN and infinities between two others changes neither of them.
    lengths = [70, 61, 75]
    g = _gen(7)
    q, k, v = (_rand(g, sum(lengths), h, dim, dtype=BF16) for h in (4, 2, 2))
    k[70:131], v[70:131] = NAN, float("inf")
    q[70:131] = NAN
    out = torch.zeros((sum(lengths), 4, dim), device="cuda", dtype=BF16)
    lse = torch.empty((sum(lengths), 4), device="cuda")
    at.prompt(ctx, q, k, v, _starts(lengths), out, lse=lse)
    for a, b in ((0, 70), (131, 206)):
        w = ref.attend(q[a:b], k[a:b], v[a:b], 0, True, 0, dim ** -0.5)
        _check_out(out[a:b], lse[a:b], [w])


def test_prompt_tokens_of_no_sequence(ctx, at):
    q, k, v = (_rand(_gen(8), 60, h, 64, dtype=F16) for h in (2, 2, 2))
    out = torch.full((60, 2, 64), 7.0, device="cuda", dtype=F16)
    starts = torch.tensor([10, 10, 40], dtype=torch.int32, device="cuda")
    at.prompt(ctx, q, k, v, starts, out)
    assert (out[:10] == 7).all() and (out[40:] == 7).all()
    w = ref.attend(q[10:40], k[10:40], v[10:40], 0, True, 0, 0.125)
    _close(out[10:40], w[0], w[2], "inner sequence")


def test_prompt_strides(ctx, at):
    g = _gen(9)
    for q, k, v in (
            # heads outermost
            tuple(_rand(g, h, 90, 64, dtype=BF16).transpose(0, 1) for h in (4, 2, 2)),
            # 2-byte aligned
            tuple(_rand(g, 90 * h * 64 + 1, dtype=BF16)[1:].view(90, h, 64) for h in (4, 2, 2)),
            # padded rows: 16-byte aligned, then not
            tuple(_rand(g, 90, h, 72, dtype=BF16)[..., :64] for h in (4, 2, 2)),
            tuple(_rand(g, 90, h, 65, dtype=BF16)[..., :64] for h in (4, 2, 2)),
            # k and v shared by all heads' groups: stride 0 over heads
            (_rand(g, 90, 4, 64, dtype=BF16),
             _rand(g, 90, 1, 64, dtype=BF16).expand(90, 2, 64),
             _rand(g, 90, 1, 64, dtype=BF16).expand(90, 2, 64))):
        out = torch.full((4, 90, 64), NAN, device="cuda", dtype=BF16).transpose(0, 1)
        lse = torch.empty((90, 4), device="cuda")
        at.prompt(ctx, q, k, v, _starts([90]), out, lse=lse)
        _check_out(out, lse, [ref.attend(q, k, v, 0, True, 0, 0.125)])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_large_scores(ctx, at, dtype):
    # Scores of hundreds: the running maximum moves a lot; weights underflow to zero.
    q, k, v = (_rand(_gen(10), 300, h, 128, dtype=dtype, size=s)
               for h, s in ((2, 6.0), (1, 6.0), (1, 1.0)))
    k[200:] *= 4
    out = torch.empty((300, 2, 128), device="cuda", dtype=dtype)
    lse = torch.empty((300, 2), device="cuda")
    at.prompt(ctx, q, k, v, _starts([300]), out, lse=lse)
    _check_out(out, lse, [ref.attend(q, k, v, 0, True, 0, 128 ** -0.5)])
    for scale in (0.0, -0.1):
        at.prompt(ctx, q, k, v, _starts([300]), out, lse=lse, scale=scale)
        _check_out(out, lse, [ref.attend(q, k, v, 0, True, 0, scale)])


class _Paged:
    """Sequences' keys and values scattered over a pool whose every other slot holds NaN."""

    def __init__(self, g, lengths, hkv, dim, page, dtype, order, spare=3):
        need = [(n + page - 1) // page for n in lengths]
        total = sum(need) + spare
        shape = (total, page, hkv, dim) if order == "slots" else (total, hkv, page, dim)
        self.k, self.v = (torch.full(shape, NAN, device="cuda", dtype=dtype) for _ in range(2))
        if order == "heads":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        perm = torch.randperm(total, device="cuda", generator=g)
        # Table entries past a sequence's pages are junk that must not be followed.
        self.table = torch.full((len(lengths), max(need + [1]) + 2), 2 ** 31 - 1, dtype=torch.int32,
                                device="cuda")
        self.keys, self.values, at = [], [], 0
        for s, n in enumerate(lengths):
            ids = perm[at:at + need[s]]
            at += need[s]
            self.table[s, :need[s]] = ids.to(torch.int32)
            kk, vv = (_rand(g, n, hkv, dim, dtype=dtype, size=1.5) for _ in range(2))
            j = torch.arange(n, device="cuda")
            self.k[ids[j // page], j % page] = kk
            self.v[ids[j // page], j % page] = vv
            self.keys.append(kk)
            self.values.append(vv)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")


CACHED = [
    # (keys, new) of each sequence, hq, hkv, dim, page, dtype, window, order
    ([(1, 1)], 1, 1, 64, 16, F16, 0, "slots"), ([(777, 1)], 8, 2, 64, 16, F16, 0, "slots"),
    ([(5, 1), (130, 1), (64, 1), (1, 1)], 8, 2, 128, 16, BF16, 0, "heads"),
    ([(2050, 1), (0, 0), (900, 1)], 32, 8, 128, 64, BF16, 0, "slots"),
    ([(300, 1)], 7, 1, 80, 32, F16, 0, "slots"), ([(129, 1), (1000, 1)], 16, 1, 96, 128, BF16, 0, "heads"),
    ([(500, 1)], 4, 4, 128, 16, F16, 100, "slots"), ([(40, 1)] * 33, 4, 2, 64, 8, BF16, 0, "slots"),
    ([(200, 2), (90, 3), (3, 3)], 4, 1, 128, 16, BF16, 0, "slots"),
    ([(300, 40), (1, 1), (1000, 100), (64, 64)], 8, 2, 128, 32, BF16, 0, "slots"),
    ([(700, 300)], 28, 4, 128, 16, F16, 0, "heads"), ([(333, 129), (50, 0), (20, 5)], 6, 6, 64, 16, BF16, 50, "slots"),
    ([(257, 17)], 5, 1, 112, 24, F16, 0, "slots"), ([(100, 20)], 4, 2, 192, 16, BF16, 0, "slots"),
    ([(100, 20), (33, 1)], 4, 2, 33, 5, F16, 9, "heads"), ([(64, 9)], 2, 1, 64, 4, F32, 0, "slots"),
    ([(77, 1)], 2, 1, 64, 1, BF16, 0, "slots"), ([(90, 1)], 160, 1, 128, 16, BF16, 0, "slots"),
    ([(6000, 30)], 8, 1, 128, 16, BF16, 0, "slots"), ([(20000, 1)], 4, 1, 128, 16, BF16, 0, "slots"),
    ([(3, 5), (0, 4), (2, 1)], 4, 2, 64, 16, F16, 0, "slots"),       # rows before the first key
    ([(10, 200)], 8, 2, 128, 16, BF16, 0, "slots"), ([(600, 500)], 2, 2, 64, 128, F16, 1, "slots"),
    ([(256, 16)], 16, 2, 64, 16, BF16, 3, "heads"), ([(4000, 8)], 16, 8, 128, 48, F16, 1500, "slots")]


@pytest.mark.parametrize("seqs,hq,hkv,dim,page,dtype,window,order", CACHED)
def test_cached(ctx, at, seqs, hq, hkv, dim, page, dtype, window, order):
    g = _gen(11)
    lengths, new = [s[0] for s in seqs], [s[1] for s in seqs]
    c = _Paged(g, lengths, hkv, dim, page, dtype, order)
    t = sum(new)
    q = _rand(g, t, hq, dim, dtype=dtype, size=1.5)
    out = torch.full((t, hq, dim), NAN, device="cuda", dtype=dtype)
    lse = torch.full((t, hq), NAN, device="cuda")
    cache, starts = at.KvCache(c.k, c.v), _starts(new)
    at.cached(ctx, q, cache, starts, c.lengths, c.table, out, max_new=max(new), lse=lse, window=window)
    torch.cuda.synchronize()
    ctx.check_device()
    wants, a = [], 0
    for s, n in enumerate(new):
        wants.append(ref.attend(q[a:a + n], c.keys[s], c.values[s], lengths[s] - n, True, window,
                                dim ** -0.5))
        a += n
    _check_out(out, lse, wants)
    again = torch.full_like(out, NAN)
    at.cached(ctx, q, cache, starts, c.lengths, c.table, again, max_new=max(new), window=window)
    assert torch.equal(out, again)
    # A larger bound on the new tokens only changes which kernel runs.
    at.cached(ctx, q, cache, starts, c.lengths, c.table, again, max_new=max(new) + 64, lse=lse,
              window=window)
    ctx.check_device()
    _check_out(again, lse, wants)


def _check_some(out, lse, seqs, every, attend):
    """Checks every `every`-th sequence (and the first and last ones) of many."""
    at = 0
    for s, n in enumerate(seqs):
        if n and (s % every == 0 or s < 3 or s >= len(seqs) - 3):
            _check_out(out[at:at + n], lse[at:at + n], [attend(s, at, n)])
        at += n
    assert at == out.shape[0] and torch.isfinite(out).all()


@pytest.mark.parametrize("count,longest,hq,hkv,dim", [(700, 40, 4, 2, 64), (150, 300, 16, 8, 128),
                                                      (33, 900, 6, 6, 80)])
def test_prompt_many_sequences(ctx, at, count, longest, hq, hkv, dim):
    # More items than CTAs: handed out by a counter that the call leaves as it found it.
    g = _gen(30)
    lengths = torch.randint(0, longest + 1, (count,), generator=torch.Generator().manual_seed(count))
    lengths = lengths.tolist()
    t = sum(lengths)
    q, k, v = (_rand(g, t, h, dim, dtype=BF16) for h in (hq, hkv, hkv))
    starts = _starts(lengths)
    out, lse = torch.full_like(q, NAN), torch.full((t, hq), NAN, device="cuda")
    for _ in range(3):
        again = torch.full_like(q, NAN)
        at.prompt(ctx, q, k, v, starts, again, lse=lse)
        if torch.isfinite(out).all():
            assert torch.equal(out, again)
        out = again
    ctx.check_device()
    _check_some(out, lse, lengths, max(1, count // 8), lambda s, a, n: ref.attend(
        q[a:a + n], k[a:a + n], v[a:a + n], 0, True, 0, dim ** -0.5))


@pytest.mark.parametrize("count,longest,chunk,hq,hkv,dim,page,window", [
    (700, 90, 1, 8, 2, 64, 16, 0), (300, 500, 1, 7, 1, 128, 16, 60), (40, 1500, 6, 32, 4, 128, 32, 0),
    (9, 3000, 90, 8, 8, 64, 128, 0), (3, 4000, 200, 28, 4, 128, 16, 900), (200, 200, 30, 4, 2, 96, 8, 0)])
def test_cached_many_sequences(ctx, at, count, longest, chunk, hq, hkv, dim, page, window):
    g, rng = _gen(31), torch.Generator().manual_seed(count)
    new = torch.randint(0, chunk + 1, (count,), generator=rng).tolist()
    lengths = [n + int(torch.randint(0, longest, (1,), generator=rng)) for n in new]
    c = _Paged(g, lengths, hkv, dim, page, F16, "slots")
    t = sum(new)
    q = _rand(g, t, hq, dim, dtype=F16)
    out, lse = torch.full_like(q, NAN), torch.full((t, hq), NAN, device="cuda")
    cache, starts = at.KvCache(c.k, c.v), _starts(new)
    at.cached(ctx, q, cache, starts, c.lengths, c.table, out, max_new=chunk, lse=lse, window=window)
    again = torch.full_like(q, NAN)
    at.cached(ctx, q, cache, starts, c.lengths, c.table, again, max_new=chunk, window=window)
    ctx.check_device()
    assert torch.equal(out, again)
    _check_some(out, lse, new, max(1, count // 8), lambda s, a, n: ref.attend(
        q[a:a + n], c.keys[s], c.values[s], lengths[s] - n, True, window, dim ** -0.5))


def test_prompt_long_split_over_the_device(ctx, at):
    # Few items of many key tiles: cut into equal shares, pieces joined; S8 and lse as well.
    g = _gen(32)
    q, k, v = (_rand(g, 3000, h, 64, dtype=BF16) for h in (2, 1, 1))
    out, lse = torch.empty_like(q), torch.empty((3000, 2), device="cuda")
    at.prompt(ctx, q, k, v, _starts([3000]), out, lse=lse)
    out8 = torch.empty((3000, 2, 64), dtype=torch.int8, device="cuda")
    at.prompt(ctx, q, k, v, _starts([3000]), at.Quantised(out8, 0.004, 2))
    rows = [0, 1, 127, 128, 500, 1023, 1024, 2047, 2500, 2998, 2999]
    for r in rows:
        w = ref.attend(q[r:r + 1], k, v, r, True, 0, 0.125)
        _check_out(out[r:r + 1], lse[r:r + 1], [w])
        _check_out(out8[r:r + 1], lse[r:r + 1], [w], 0.004, 2)


def test_cached_not_causal(ctx, at):
    c = _Paged(_gen(12), [150, 7], 2, 64, 16, BF16, "slots")
    q = _rand(_gen(13), 12, 4, 64, dtype=BF16)
    for bound in (10, 80):
        out = torch.full((12, 4, 64), NAN, device="cuda", dtype=BF16)
        lse = torch.empty((12, 4), device="cuda")
        at.cached(ctx, q, at.KvCache(c.k, c.v), _starts([10, 2]), c.lengths, c.table, out, bound,
                  lse=lse, causal=False)
        wants = [ref.attend(q[a:b], c.keys[s], c.values[s], 0, False, 0, 0.125)
                 for s, (a, b) in enumerate(((0, 10), (10, 12)))]
        _check_out(out, lse, wants)


@pytest.mark.parametrize("bound", [1, 40])
def test_cached_s8_output(ctx, at, bound):
    c = _Paged(_gen(14), [600, 33, 1200], 2, 128, 16, F16, "slots")
    q = _rand(_gen(15), 3, 8, 128, dtype=F16, size=2.0)
    out = torch.full((3, 8, 128), 55, device="cuda", dtype=torch.int8)
    lse = torch.empty((3, 8), device="cuda")
    at.cached(ctx, q, at.KvCache(c.k, c.v), _starts([1, 1, 1]), c.lengths, c.table,
              at.Quantised(out, 0.005, 3), bound, lse=lse)
    wants = [ref.attend(q[s:s + 1], c.keys[s], c.values[s], n - 1, True, 0, 128 ** -0.5)
             for s, n in enumerate((600, 33, 1200))]
    _check_out(out, lse, wants, 0.005, 3)


@pytest.mark.parametrize("bound", [1, 40])
def test_cached_window_skips_dropped_pages(ctx, at, bound):
    # Pages wholly before the window may have been given away: their entries are junk.
    c = _Paged(_gen(16), [1000], 2, 64, 16, BF16, "slots")
    first = (1000 - 200) // 16
    c.table[0, :first] = -1
    c.k[c.table[0, first].long(), : (1000 - 200) % 16] = NAN
    c.v[c.table[0, first].long(), : (1000 - 200) % 16] = float("inf")
    q = _rand(_gen(17), 1, 4, 64, dtype=BF16)
    out = torch.empty((1, 4, 64), device="cuda", dtype=BF16)
    lse = torch.empty((1, 4), device="cuda")
    at.cached(ctx, q, at.KvCache(c.k, c.v), _starts([1]), c.lengths, c.table, out, bound, lse=lse,
              window=200)
    _check_out(out, lse, [ref.attend(q, c.keys[0], c.values[0], 999, True, 200, 0.125)])


@pytest.mark.parametrize("bound", [1, 40])
def test_cached_offsets_past_32_bits(ctx, at, bound):
    # A pool of 2^32 + elements: the last pages' offsets do not fit 32 bits.
    pages, page, hkv, dim = 2100, 128, 128, 128
    k = torch.empty((pages, page, hkv, dim), dtype=F16, device="cuda")
    v = torch.empty_like(k)
    ids = torch.tensor([pages - 1, 2, pages - 2], device="cuda")
    g = _gen(18)
    kk, vv = (_rand(g, 300, hkv, dim, dtype=F16) for _ in range(2))
    j = torch.arange(300, device="cuda")
    k[ids[j // page], j % page], v[ids[j // page], j % page] = kk, vv
    q = _rand(g, 1, hkv, dim, dtype=F16)
    out, lse = torch.empty_like(q), torch.empty((1, hkv), device="cuda")
    at.cached(ctx, q, at.KvCache(k, v), _starts([1]), torch.tensor([300], dtype=torch.int32, device="cuda"),
              ids.to(torch.int32)[None].contiguous(), out, bound, lse=lse)
    _check_out(out, lse, [ref.attend(q, kk, vv, 299, True, 0, dim ** -0.5)])


def test_calls_on_two_streams_share_a_context(ctx, at):
    c = _Paged(_gen(19), [9000], 1, 128, 16, BF16, "slots")
    cache, starts = at.KvCache(c.k, c.v), _starts([1])
    qs = [_rand(_gen(20 + i), 1, 4, 128, dtype=BF16) for i in range(8)]
    outs = [torch.empty_like(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, q in enumerate(qs):
            at.cached(ctx, q, cache, starts, c.lengths, c.table, outs[i], 1,
                      stream=streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    for q, o in zip(qs, outs):
        w = ref.attend(q, c.keys[0], c.values[0], 8999, True, 0, 128 ** -0.5)
        _close(o, w[0], w[2], "two streams")


@pytest.mark.parametrize("bound", [1, 40])
def test_cached_in_a_graph(ctx, at, bound):
    c = _Paged(_gen(21), [5000, 70], 2, 128, 16, BF16, "slots")
    q = _rand(_gen(22), 2, 8, 128, dtype=BF16)
    out = torch.zeros_like(q)
    cache, starts = at.KvCache(c.k, c.v), _starts([1, 1])
    args = (ctx, q, cache, starts, c.lengths, c.table, out, bound)
    s = torch.cuda.Stream()
    at.cached(*args, stream=s.cuda_stream)
    torch.cuda.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        at.cached(*args, stream=s.cuda_stream)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_first_call_of_a_context_cannot_be_captured(at):
    from pspml import capi
    c = _Paged(_gen(24), [60], 1, 64, 16, BF16, "slots")
    q = _rand(_gen(25), 1, 2, 64, dtype=BF16)
    out = torch.zeros_like(q)
    with capi.Context(0) as own:
        args = (own, q, at.KvCache(c.k, c.v), _starts([1]), c.lengths, c.table, out, 1)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            with pytest.raises(capi.PspmlError, match="UNSUPPORTED.*captured"):
                at.cached(*args, stream=s.cuda_stream)
        at.cached(*args, stream=s.cuda_stream)
        torch.cuda.synchronize()
        w = ref.attend(q, c.keys[0], c.values[0], 59, True, 0, 0.125)
        _close(out, w[0], w[2], "after a refused capture")


def test_python_refusals(ctx, at):
    q = torch.zeros((4, 2, 64), device="cuda", dtype=F16)
    starts = _starts([4])
    with pytest.raises(ValueError, match="dtype"):
        at.prompt(ctx, q.double(), q, q, starts, q.clone())
    with pytest.raises(ValueError, match="cpu"):
        at.prompt(ctx, q.cpu(), q, q, starts, q.clone())
    with pytest.raises(ValueError, match="tokens"):
        at.prompt(ctx, q, q[:3], q[:3], starts, q.clone())
    with pytest.raises(ValueError, match="starts"):
        at.prompt(ctx, q, q, q, starts.long(), q.clone())
    with pytest.raises(ValueError, match="contiguous"):
        at.prompt(ctx, q.transpose(1, 2), q, q, starts, q.clone())
    with pytest.raises(ValueError, match="pools"):
        at.KvCache(torch.zeros(2, 4, 1, 8), torch.zeros(2, 5, 1, 8))
    r = at.Rotary(ctx, 64)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="positions"):
        at.rotary_apply(r, pos[:3], q, q)
    from pspml import capi
    with pytest.raises(capi.PspmlError, match="INVALID_ARG"):
        at.rotary_apply(at.Rotary(ctx, 32), pos, q, q.clone())
    with pytest.raises(capi.PspmlError, match="in-place"):
        at.rotary_apply(r, pos, q, q.as_strided((4, 2, 64), (64, 256, 1)))


def test_rotary_outlives_its_context(ctx, at):
    from pspml import capi
    with capi.Context(0) as other:
        r = at.Rotary(other, 64)
    q = _rand(_gen(23), 3, 2, 64)
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    out, want = torch.empty_like(q), torch.empty_like(q)
    at.rotary_apply(r, pos, q, out)
    r.close()
    at.rotary_apply(at.Rotary(ctx, 64), pos, q, want)  # no error is left behind either
    assert torch.equal(out, want)


def test_nothing_to_do(ctx, at):
    empty = torch.zeros((0, 2, 64), device="cuda", dtype=F16)
    at.prompt(ctx, empty, empty, empty, _starts([0]), empty.clone())
    at.rotary_apply(at.Rotary(ctx, 64), torch.zeros(0, dtype=torch.int32, device="cuda"), empty,
                    empty.clone())
    q = torch.full((3, 2, 64), 1.0, device="cuda", dtype=F16)
    out = torch.full_like(q, 5.0)
    at.prompt(ctx, q, q, q, torch.zeros(1, dtype=torch.int32, device="cuda"), out)
    torch.cuda.synchronize()
    assert (out == 5).all()


# What a key holds must not reach rows that do not see it, in the tiles of the
# rows that do: (token from the end, column or None for all, value, in k or v).
POISON = [(1, 3, NAN, "v"), (9, None, math.inf, "v"), (70, 7, -math.inf, "v"), (71, 7, NAN, "v"),
          (190, 1, NAN, "v"), (2, None, NAN, "k")]


def _check_poisoned(out, lse, want, scale8=None, zero8=0):
    """Finite where the formula is finite, and to the usual tolerance; not finite where it is
    not."""
    o, l, tol_o, tol_l = want
    fine = torch.isfinite(o)
    assert not fine.all()
    if scale8 is None:
        assert not torch.isfinite(out[~fine]).any()
    if not fine.any():
        pass
    elif scale8 is None:
        _close(out[fine], o[fine], tol_o[fine], "rows that do not see the bad keys")
    else:
        exact = (o[fine] / scale8 + zero8).clamp(-128, 127)
        _close(out[fine], exact, 0.5 + tol_o[fine] / scale8 + 1e-3, "S8")
    seen = torch.isnan(l)
    _close_lse(lse[~seen], l[~seen], tol_l[~seen])
    assert torch.isnan(lse[seen]).all()


def _poison(k, v, column_limit, deepest=1000):
    for back, column, value, where in POISON:
        if back <= min(k.shape[0], deepest):
            x = (k if where == "k" else v)[k.shape[0] - back]
            x[:, slice(None) if column is None else min(column, column_limit)] = value


@pytest.mark.parametrize("tokens,hq,hkv,dim,dtype,causal_window", [
    (300, 4, 2, 128, BF16, 0), (257, 8, 1, 64, F16, 0), (12, 3, 1, 64, BF16, 0),
    (700, 6, 2, 80, BF16, 130), (129, 2, 2, 96, F16, 3), (2600, 1, 1, 128, BF16, 0),
    (1500, 40, 40, 64, F16, 64), (500, 4, 2, 192, BF16, 0)])
def test_prompt_masked_keys_hold_nan(ctx, at, tokens, hq, hkv, dim, dtype, causal_window):
    g = _gen(40)
    q, k, v = (_rand(g, tokens, h, dim, dtype=dtype) for h in (hq, hkv, hkv))
    _poison(k, v, dim - 1)
    out, lse = torch.zeros_like(q), torch.zeros((tokens, hq), device="cuda")
    out8 = torch.zeros((tokens, hq, dim), dtype=torch.int8, device="cuda")
    at.prompt(ctx, q, k, v, _starts([tokens]), out, lse=lse, window=causal_window)
    at.prompt(ctx, q, k, v, _starts([tokens]), at.Quantised(out8, 0.02, -3), window=causal_window)
    ctx.check_device()
    first = max(0, tokens - 400)          # the rows near the bad keys, and a few before
    rows = [0] + list(range(max(1, first), tokens)) if tokens > 1 else [0]
    parts = [ref.attend(q[r:r + 1], k, v, r, True, causal_window, dim ** -0.5) for r in rows]
    want = [torch.cat(x) for x in zip(*parts)]
    _check_poisoned(out[rows], lse[rows], want)
    _check_poisoned(out8[rows], lse[rows], want, 0.02, -3)


@pytest.mark.parametrize("bound", [4, 80])
@pytest.mark.parametrize("deepest", [2, 1000])  # 1000: keys that all rows see as well
@pytest.mark.parametrize("lengths,new,hq,hkv,dim,page,dtype,window", [
    ([600, 70], [4, 4], 8, 4, 128, 16, BF16, 0), ([90, 300, 5, 2000], [4, 3, 4, 2], 4, 1, 64, 8, F16, 0),
    ([3, 40], [4, 2], 2, 1, 80, 16, BF16, 0), ([5000, 1200], [4, 4], 4, 2, 128, 32, F16, 3),
    ([900], [4], 16, 4, 96, 16, BF16, 200)])
def test_cached_masked_keys_hold_nan(ctx, at, bound, deepest, lengths, new, hq, hkv, dim, page, dtype,
                                     window):
    # Also rows that see no key at all beside rows that do ([3, 40] with 4 new tokens).
    c = _Paged(_gen(41), lengths, hkv, dim, page, dtype, "slots")
    for s, n in enumerate(lengths):
        _poison(c.keys[s], c.values[s], dim - 1, deepest)
        j = torch.arange(n, device="cuda")
        ids = c.table[s].long()[j // page]
        c.k[ids, j % page], c.v[ids, j % page] = c.keys[s], c.values[s]
    q = _rand(_gen(42), sum(new), hq, dim, dtype=dtype)
    out, lse = torch.zeros_like(q), torch.zeros((sum(new), hq), device="cuda")
    at.cached(ctx, q, at.KvCache(c.k, c.v), _starts(new), c.lengths, c.table, out, bound, lse=lse,
              window=window)
    ctx.check_device()
    a, parts = 0, []
    for s, n in enumerate(new):
        parts.append(ref.attend(q[a:a + n], c.keys[s], c.values[s], lengths[s] - n, True, window,
                                dim ** -0.5))
        a += n
    want = [torch.cat(x) for x in zip(*parts)]
    assert deepest > 2 or torch.isfinite(want[0]).any()
    _check_poisoned(out, lse, want)


@pytest.mark.parametrize("dim,hq,hkv", [(128, 8, 2), (64, 3, 3)])
def test_all_values_nan_or_infinite(ctx, at, dim, hq, hkv):
    # Every row sees a bad key: nothing is finite, and nothing takes long.
    q, k = (_rand(_gen(43), 4000, h, dim, dtype=BF16) for h in (hq, hkv))
    out = torch.zeros_like(q)
    for value in (NAN, math.inf):
        at.prompt(ctx, q, k, torch.full_like(k, value), _starts([4000]), out)
        ctx.check_device()
        assert not torch.isfinite(out).any()
