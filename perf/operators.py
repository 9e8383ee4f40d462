"""Timed cases of the attention operators: rotary positions, the append to a
paged key/value cache, attention over whole prompts and attention of new
tokens over the cache.

``run`` computes a case with elementary torch operations in 32 bits, or, with
``own`` set, through this package's entry points.
"""
import math
import random
import sys

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "s8": torch.int8}
_handles = {}


def _package():
    """The package's modules and one context on the current GPU, as a program keeps them."""
    if "ctx" not in _handles:
        if "psp-ml_b200" not in sys.path:
            sys.path.insert(0, "psp-ml_b200")
        from pspml import attention, capi

        _handles["attention"] = attention
        _handles["capi"] = capi
        _handles["ctx"] = capi.Context(torch.cuda.current_device())
    return _handles["attention"], _handles["capi"], _handles["ctx"]


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One decoding step of eight requests: q and k sliced from one projection's output.
        dict(name="rotary_step", op="rotary", tokens=8, hq=32, hkv=8, dim=128, rot=128,
             layout="half", dtype="bf16", base=500000.0, scaling="parts", farthest=100000),
        # A long prompt through a network that rotates half of each head, interleaved pairs.
        dict(name="rotary_prompt", op="rotary", tokens=16384, hq=32, hkv=8, dim=128, rot=64,
             layout="interleaved", dtype="f16", base=10000.0, scaling="none", farthest=16384),
        # The cache append of a decoding batch.
        dict(name="append_step", op="append", tokens=64, hq=32, hkv=8, dim=128, rot=128,
             layout="half", dtype="bf16", base=10000.0, scaling="linear", farthest=32768,
             page=16, pages=4096, order="slots"),
        # A prompt straight from int8 projections: dequantised, rotated and appended in one pass.
        dict(name="append_prompt_s8", op="append", tokens=8191, hq=28, hkv=4, dim=128, rot=128,
             layout="half", dtype="s8", base=1000000.0, scaling="none", farthest=65536,
             page=64, pages=160, order="heads"),
        # The first, short prompt of an interactive session on a small network.
        dict(name="prompt_short", op="prompt", seqs=1, longest=37, mix=1, hq=8, hkv=2, dim=64,
             dtype="f16", window=0),
        # Packed prompts of unlike lengths.
        dict(name="prompt_packed", op="prompt", seqs=17, longest=2048, mix=2, hq=32, hkv=8, dim=128,
             dtype="bf16", window=0),
        # Packed prompts of a network with one key head a query head, an 80-wide head, a window.
        dict(name="prompt_window", op="prompt", seqs=5, longest=4001, mix=3, hq=20, hkv=20, dim=80,
             dtype="f16", window=1000),
        # A whole document.
        dict(name="prompt_long", op="prompt", seqs=1, longest=16384, mix=4, hq=32, hkv=8, dim=128,
             dtype="bf16", window=0),
        # One token of one short conversation.
        dict(name="step_single", op="cached", seqs=1, longest=777, chunk=1, mix=5, hq=8, hkv=2,
             dim=64, dtype="f16", window=0, page=16, order="slots"),
        # One token of each of 64 conversations of unlike lengths.
        dict(name="step_batch", op="cached", seqs=64, longest=8192, chunk=1, mix=6, hq=32, hkv=8,
             dim=128, dtype="bf16", window=0, page=16, order="slots"),
        # One token over a very long document.
        dict(name="step_long", op="cached", seqs=1, longest=131077, chunk=1, mix=7, hq=32, hkv=8,
             dim=128, dtype="bf16", window=0, page=64, order="heads"),
        # Prompt chunks and single tokens in one batch over their caches.
        dict(name="chunk_mixed", op="cached", seqs=6, longest=12000, chunk=512, mix=8, hq=28, hkv=4,
             dim=128, dtype="bf16", window=0, page=32, order="slots"),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "prompt", "cached", "cached"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([64, 80, 96, 128, 128])
    case = dict(op=op, hq=hkv * group, hkv=hkv, dim=dim)
    if op in ("rotary", "append"):
        case.update(tokens=_between(rng, 1, 16384), rot=rng.choice([dim, dim, dim // 2]),
                    layout=rng.choice(["half", "interleaved"]),
                    dtype=rng.choice(["f16", "bf16", "s8"]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]),
                    scaling=rng.choice(["none", "linear", "parts"]),
                    farthest=_between(rng, 1000, 200000))
        if op == "append":
            page = rng.choice([16, 32, 64, 128])
            case.update(page=page, pages=case["tokens"] // page + rng.randint(2, 100),
                        order=rng.choice(["slots", "heads"]))
        return case
    case.update(dtype=rng.choice(["f16", "bf16"]), mix=rng.randint(10, 10 ** 6),
                window=rng.choice([0, 0, 0, rng.randint(1, 2000)]))
    if op == "prompt":
        longest = _between(rng, 1, 8192)
        case.update(seqs=_between(rng, 1, max(1, min(40, 16384 // longest))), longest=longest)
    else:
        chunk = rng.choice([1, 1, 1, _between(rng, 2, 16), _between(rng, 17, 1024)])
        longest = _between(rng, max(16, chunk), 65536)
        case.update(seqs=_between(rng, 1, max(1, min(128, 262144 // longest))), longest=longest,
                    chunk=chunk, page=rng.choice([16, 32, 64, 128]),
                    order=rng.choice(["slots", "heads"]))
    return case


def _lengths(case):
    """(keys, new tokens) of each sequence; the first is the longest."""
    rng = random.Random(case["mix"])
    keys, new = [], []
    for s in range(case["seqs"]):
        if case["op"] == "prompt":
            n = case["longest"] if s == 0 else _between(rng, 1, case["longest"])
            keys.append(n)
            new.append(n)
        else:
            n = case["chunk"] if s == 0 else _between(rng, 1, case["chunk"])
            new.append(n)
            keys.append(case["longest"] if s == 0 else rng.randint(n, max(n, case["longest"])))
    return keys, new


def _pairs(case):
    """Query-key pairs of one head that the masks keep, over the whole case."""
    total = 0
    for length, n in zip(*_lengths(case)):
        first, w = length - n, case["window"]
        if w == 0:
            total += n * first + n * (n + 1) // 2
        else:
            full = max(0, min(n, w - first))  # rows that still see every key before them
            total += full * first + full * (full + 1) // 2 + (n - full) * w
    return total


def _keys_read(case):
    total = 0
    for length, n in zip(*_lengths(case)):
        total += min(length, n + case["window"] - 1) if case["window"] else length
    return total


def work(case):
    d, hq, hkv = case["dim"], case["hq"], case["hkv"]
    if case["op"] in ("rotary", "append"):
        size = 1 if case["dtype"] == "s8" else 2
        heads = hq + hkv * (2 if case["op"] == "append" else 1)
        per_token = heads * d * (size + 2) + (12 if case["op"] == "append" else 4)
        return {"bytes": case["tokens"] * per_token,
                "flops": 3 * case["tokens"] * (hq + hkv) * case["rot"]}
    rows = sum(_lengths(case)[1])
    return {"bytes": 2 * d * (2 * rows * hq + 2 * _keys_read(case) * hkv),
            "flops": 4 * d * hq * _pairs(case)}


# ------------------------------------------------------------------ inputs

def _frequencies(case):
    """Angles a token (float64): the case's base, positions scaled evenly or, by parts, only
    those that turn less than four times over the original length."""
    rot = case["rot"]
    f = case["base"] ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        f = f / 4.0
    elif case["scaling"] == "parts":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = keep * f + (1 - keep) * f / 8.0
    return f


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    d, hq, hkv = case["dim"], case["hq"], case["hkv"]
    state = {"case": case}

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, device="cuda", generator=g, dtype=dtype)

    if case["op"] in ("rotary", "append"):
        t, out = case["tokens"], torch.float16 if case["dtype"] == "s8" else _DTYPES[case["dtype"]]
        if case["dtype"] == "s8":
            x = torch.randint(-128, 128, (t, hq + 2 * hkv, d), device="cuda", generator=g,
                              dtype=torch.int8)
            state.update(scale=0.03125, zero=-3)
        else:
            x = normal(t, hq + 2 * hkv, d, dtype=out)
            x[:, :, ::13] *= 4
        first = torch.randint(0, max(1, case["farthest"] - t), (1,), device="cuda", generator=g)
        if case["op"] == "append" and t <= 128:  # a token of each of t sequences
            pos = torch.randint(0, case["farthest"], (t,), device="cuda", generator=g)
        else:
            pos = first + torch.arange(t, device="cuda")
        state.update(q=x[:, :hq], k=x[:, hq:hq + hkv], v=x[:, hq + hkv:],
                     positions=pos.to(torch.int32),
                     q_out=torch.empty((t, hq, d), device="cuda", dtype=out))
        if case["op"] == "rotary":
            state["k_out"] = torch.empty((t, hkv, d), device="cuda", dtype=out)
        else:
            state.update(_pools(case, case["pages"], normal, out))
            total = case["pages"] * case["page"]
            state["slots"] = torch.randperm(total, device="cuda", generator=g)[:t]
            if t > 128:  # a prompt fills whole pages in a random order
                pages = torch.randperm(case["pages"], device="cuda", generator=g)
                i = torch.arange(t, device="cuda")
                state["slots"] = pages[i // case["page"]] * case["page"] + i % case["page"]
        if own:
            attention, capi, ctx = _package()
            factor = {"none": 1.0, "linear": 4.0, "parts": 8.0}[case["scaling"]]
            state["rotary"] = attention.Rotary(
                ctx, head_dim=d, rot_dim=case["rot"], layout=case["layout"], base=case["base"],
                scaling=case["scaling"], factor=factor, original_len=8192, low=1.0, high=4.0)
            if case["op"] == "append":
                state["cache"] = attention.KvCache(state["k_pool"], state["v_pool"])
        else:
            span = case["farthest"] + t
            angles = torch.arange(span, dtype=torch.float64, device="cuda")[:, None] * \
                _frequencies(case).cuda()
            state.update(cos=angles.cos().float(), sin=angles.sin().float())
        return state

    dtype = _DTYPES[case["dtype"]]
    keys, new = _lengths(case)
    rows = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state.update(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 out=torch.empty((rows, hq, d), device="cuda", dtype=dtype))
    if case["op"] == "prompt":
        x = normal(rows, hq + 2 * hkv, d, dtype=dtype)
        x[:, :hq + hkv, ::13] *= 2
        state.update(q=x[:, :hq], k=x[:, hq:hq + hkv], v=x[:, hq + hkv:])
        return state
    q = normal(rows, hq, d, dtype=dtype)
    q[:, :, ::13] *= 2
    page = case["page"]
    need = [(n + page - 1) // page for n in keys]
    total = sum(need) + 3
    state.update(q=q, **_pools(case, total, normal, dtype))
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros((len(keys), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    state.update(table=table, keys=torch.tensor(keys, dtype=torch.int32, device="cuda"))
    if own:
        attention, capi, ctx = _package()
        state["cache"] = attention.KvCache(state["k_pool"], state["v_pool"])
    return state


def _pools(case, pages, normal, dtype):
    """Key and value pools [pages][page][heads][dim]; "heads" keeps a page's slots of one head
    together in memory."""
    pools = []
    for _ in range(2):
        if case["order"] == "heads":
            p = normal(pages, case["hkv"], case["page"], case["dim"], dtype=dtype).transpose(1, 2)
        else:
            p = normal(pages, case["page"], case["hkv"], case["dim"], dtype=dtype)
        pools.append(p)
    return {"k_pool": pools[0], "v_pool": pools[1]}


# ------------------------------------------------------------------- passes

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state["case"]
    attention, _, ctx = _package()
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] in ("rotary", "append"):
        q, k, v = state["q"], state["k"], state["v"]
        if case["dtype"] == "s8":
            q, k, v = (attention.Quantised(x, state["scale"], state["zero"]) for x in (q, k, v))
        if case["op"] == "rotary":
            attention.rotary_apply(state["rotary"], state["positions"], q, state["q_out"], k,
                                   state["k_out"], stream=stream)
            return state["q_out"], state["k_out"]
        attention.rotary_append(state["rotary"], state["positions"], state["slots"], q,
                                state["q_out"], k, v, state["cache"], stream=stream)
        return state["q_out"], state["k_pool"], state["v_pool"]
    if case["op"] == "prompt":
        attention.prompt(ctx, state["q"], state["k"], state["v"], state["starts"], state["out"],
                         window=case["window"], stream=stream)
    else:
        attention.cached(ctx, state["q"], state["cache"], state["starts"], state["keys"],
                         state["table"], state["out"], max_new=case["chunk"],
                         window=case["window"], stream=stream)
    return state["out"]


def _rotate(x, cos, sin, rot, layout):
    head, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    return torch.cat((turned, rest), dim=-1)


def _attend(q, k, v, first, window):
    """Causal attention of q [rows][hq][dim], whose first row sits at position `first`, over
    k and v [keys][hkv][dim], all in 32 bits."""
    rows, hq, d = q.shape
    keys, hkv, _ = k.shape
    group = hq // hkv
    kt, vt = k.permute(1, 2, 0), v.permute(1, 0, 2)
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // (hq * keys))
    for a in range(0, rows, step):
        b = min(rows, a + step)
        end = first + b
        at = torch.arange(first + a, end, device=q.device)[:, None]
        key = torch.arange(end, device=q.device)[None]
        hidden = key > at
        if window:
            hidden |= key <= at - window
        part = q[a:b].reshape(b - a, hkv, group, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        s = torch.bmm(part, kt[:, :, :end]).view(hkv, group, b - a, end) * (1.0 / math.sqrt(d))
        s.masked_fill_(hidden, -math.inf)
        top = s.amax(dim=-1, keepdim=True)
        p = torch.exp(s - top)
        o = torch.bmm(p.view(hkv, -1, end), vt[:, :end]) / p.sum(dim=-1).view(hkv, -1, 1)
        out[a:b] = o.view(hkv, group, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d)
    return out


def _run_plain(state):
    case = state["case"]
    if case["op"] in ("rotary", "append"):
        values = [state[n] for n in "qkv"]
        if case["dtype"] == "s8":
            values = [(x.float() - state["zero"]) * state["scale"] for x in values]
        q, k, v = (x.float() for x in values)
        at = state["positions"].long()
        cos, sin = state["cos"][at][:, None], state["sin"][at][:, None]
        state["q_out"].copy_(_rotate(q, cos, sin, case["rot"], case["layout"]))
        k = _rotate(k, cos, sin, case["rot"], case["layout"])
        if case["op"] == "rotary":
            state["k_out"].copy_(k)
            return state["q_out"], state["k_out"]
        page, slot = state["slots"] // case["page"], state["slots"] % case["page"]
        for pool, x in ((state["k_pool"], k), (state["v_pool"], v)):
            pool[page, slot] = x.to(pool.dtype)
        return state["q_out"], state["k_pool"], state["v_pool"]
    keys, new = _lengths(case)
    at = 0
    for s, (length, n) in enumerate(zip(keys, new)):
        if case["op"] == "prompt":
            k, v = state["k"][at:at + n], state["v"][at:at + n]
        else:
            pages = state["table"][s, :(length + case["page"] - 1) // case["page"]].long()
            k, v = (state[p][pages].flatten(0, 1)[:length] for p in ("k_pool", "v_pool"))
        o = _attend(state["q"][at:at + n].float(), k.float(), v.float(), length - n,
                    case["window"])
        state["out"][at:at + n] = o.to(state["out"].dtype)
        at += n
    return state["out"]


# -------------------------------------------------------------------- exact

def exact(case, seed):
    """What run returns, from the definitions in 64 bits."""
    state = prepare(case, seed)
    if case["op"] in ("rotary", "append"):
        return _exact_rotary(case, state)
    keys, new = _lengths(case)
    d, group = case["dim"], case["hq"] // case["hkv"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (length, n) in enumerate(zip(keys, new)):
        for h in range(case["hkv"]):
            if case["op"] == "prompt":
                k, v = state["k"][at:at + n, h].double(), state["v"][at:at + n, h].double()
            else:
                j = torch.arange(length, device="cuda")
                page, slot = state["table"][s].long()[j // case["page"]], j % case["page"]
                k = state["k_pool"][page, slot, h].double()
                v = state["v_pool"][page, slot, h].double()
            for head in range(h * group, (h + 1) * group):
                for r in range(0, n, 2048):
                    q = state["q"][at + r:at + min(n, r + 2048), head].double()
                    place = length - n + r + torch.arange(len(q), device="cuda")
                    low = max(0, int(place[0]) - case["window"] + 1) if case["window"] else 0
                    high = int(place[-1]) + 1
                    j = torch.arange(low, high, device="cuda")
                    seen = j[None] <= place[:, None]
                    if case["window"]:
                        seen &= j[None] > place[:, None] - case["window"]
                    scores = (q @ k[low:high].T / d ** 0.5).where(seen, -math.inf)
                    out[at + r:at + r + len(q), head] = scores.softmax(dim=1) @ v[low:high]
        at += n
    return out


def _exact_rotary(case, state):
    def value(x):
        x = x.double()
        return state["scale"] * (x - state["zero"]) if case["dtype"] == "s8" else x

    rot = case["rot"]
    angle = state["positions"].double()[:, None] * _frequencies(case).cuda()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotated(x):
        x = value(x).clone()
        if case["layout"] == "half":
            first, second = slice(0, rot // 2), slice(rot // 2, rot)
        else:
            first, second = slice(0, rot, 2), slice(1, rot, 2)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    if case["op"] == "rotary":
        return rotated(state["q"]), rotated(state["k"])
    k_pool, v_pool = state["k_pool"].double(), state["v_pool"].double()
    page, slot = state["slots"] // case["page"], state["slots"] % case["page"]
    k_pool[page, slot] = rotated(state["k"])
    v_pool[page, slot] = value(state["v"])
    return rotated(state["q"]), k_pool, v_pool
