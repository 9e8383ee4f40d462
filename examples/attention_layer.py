"""One attention layer of an int8 decoder network, prompts first, then tokens.

The projections are the framework's int8 fully connected op; between them run
the rotary + cache append (which takes the int8 projection as it is), attention
over the packed prompts or over the paged cache, and the rounding of its
output back to the int8 that the next projection reads.  Activations stay int8
from one projection to the other; the cache and the sums are F16 and F32.

    python examples/attention_layer.py
"""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "psp-ml_b200"))

import ctypes

import torch

from pspml import attention, capi, netspec


class Projection:
    """An int8 fully connected op: real = scale * q on both sides, zero point 0."""

    def __init__(self, ctx, n_in, n_out, scale_in, scale_out, seed):
        g = torch.Generator().manual_seed(seed)
        scale_w = 1.0 / (40.0 * n_in ** 0.5)
        m, shift = netspec.quantize_multiplier(scale_in * scale_w / scale_out)
        self.ctx, self.n_out = ctx, n_out
        self.filter = torch.randint(-127, 128, (n_out, n_in), generator=g, dtype=torch.int8).cuda()
        self.mult = torch.full((n_out,), m, dtype=torch.int32, device="cuda")
        self.shift = torch.full((n_out,), shift, dtype=torch.int32, device="cuda")
        self.desc = capi.OpDesc(kind=capi.OP_FULLY_CONNECTED, in_h=1, in_w=1, in_c=n_in, out_h=1,
                                out_w=1, out_c=n_out, kernel_h=1, kernel_w=1, stride_h=1,
                                stride_w=1, act_min=-128, act_max=127)

    def __call__(self, x, stream):
        out = torch.empty((x.shape[0], self.n_out), dtype=torch.int8, device="cuda")
        capi.call("pspml_fully_connected_s8", self.ctx.handle, ctypes.byref(self.desc), x.shape[0],
                  x.data_ptr(), self.filter.data_ptr(), None, self.mult.data_ptr(),
                  self.shift.data_ptr(), out.data_ptr(), stream)
        return out


class AttentionLayer:
    """q_heads query heads over kv_heads key heads, with a cache of `pages` pages."""

    def __init__(self, ctx, q_heads=8, kv_heads=2, dim=64, pages=64, page_size=16, seed=0):
        self.ctx, self.q_heads, self.kv_heads, self.dim = ctx, q_heads, kv_heads, dim
        self.width = q_heads * dim
        self.scale_in, self.scale_qkv, self.scale_attn = 0.02, 0.03, 0.01
        self.qkv = Projection(ctx, self.width, (q_heads + 2 * kv_heads) * dim, self.scale_in,
                              self.scale_qkv, seed)
        self.out = Projection(ctx, self.width, self.width, self.scale_attn, self.scale_in, seed + 1)
        self.rotary = attention.Rotary(ctx, dim, scaling="parts", factor=4.0, original_len=256)
        pool = torch.zeros((2, pages, page_size, kv_heads, dim), dtype=torch.float16, device="cuda")
        self.cache = attention.KvCache(pool[0], pool[1])
        self.page_size, self.free = page_size, list(range(pages))[::-1]
        self.tables, self.lengths = [], []

    def add_sequence(self, most_tokens):
        need = (most_tokens + self.page_size - 1) // self.page_size
        if need > len(self.free):
            raise ValueError("the cache has no room for the sequence")
        self.tables.append([self.free.pop() for _ in range(need)])
        self.lengths.append(0)

    def __call__(self, x, new):
        """x: int8 [sum(new)][width], new[s] tokens of each sequence in turn.  Appends them to
        the cache and returns (attention output, layer output), both int8 [sum(new)][width]."""
        stream = torch.cuda.current_stream().cuda_stream
        positions, slots, starts, prompts = [], [], [0], True
        for s, n in enumerate(new):
            for p in range(self.lengths[s], self.lengths[s] + n):
                positions.append(p)
                slots.append(self.tables[s][p // self.page_size] * self.page_size +
                             p % self.page_size)
            prompts &= self.lengths[s] == 0
            self.lengths[s] += n
            starts.append(starts[-1] + n)

        def ints(values, dtype=torch.int32):
            return torch.tensor(values, dtype=dtype).cuda()

        t, dim, hq, hkv = len(positions), self.dim, self.q_heads, self.kv_heads
        h = self.qkv(x, stream).view(t, hq + 2 * hkv, dim)
        q8, k8, v8 = (attention.Quantised(part, self.scale_qkv)
                      for part in (h[:, :hq], h[:, hq:hq + hkv], h[:, hq + hkv:]))
        q = torch.empty((t, hq, dim), dtype=torch.float16, device="cuda")
        attention.rotary_append(self.rotary, ints(positions), ints(slots, torch.int64), q8, q, k8,
                                v8, self.cache, stream=stream)
        mixed = torch.empty((t, hq, dim), dtype=torch.int8, device="cuda")
        o = attention.Quantised(mixed, self.scale_attn)
        if prompts:
            # Nothing cached before: the prompts' own keys are read packed, turned by the same
            # call as q (k goes to the cache and, here, to a packed copy).
            k = torch.empty((t, hkv, dim), dtype=torch.float16, device="cuda")
            attention.rotary_apply(self.rotary, ints(positions), k8, k, stream=stream)
            v = (v8.tensor.float() * self.scale_qkv).half()
            attention.prompt(self.ctx, q, k, v, ints(starts), o, stream=stream)
        else:
            most = max(len(table) for table in self.tables)
            table = ints([row + [0] * (most - len(row)) for row in self.tables])
            attention.cached(self.ctx, q, self.cache, ints(starts), ints(self.lengths), table, o,
                             max_new=max(new), stream=stream)
        mixed = mixed.view(t, self.width)
        return mixed, self.out(mixed, stream)


def main():
    torch.manual_seed(1)
    lengths, steps = [37, 5, 120], 6
    with capi.Context(0) as ctx:
        layer, whole = AttentionLayer(ctx), AttentionLayer(ctx)
        for n in lengths:
            layer.add_sequence(n + steps)
            whole.add_sequence(n + steps)
        x = [torch.randint(-127, 128, (n + steps, layer.width), dtype=torch.int8, device="cuda")
             for n in lengths]
        parts = [layer(torch.cat([r[:n] for r, n in zip(x, lengths)]), lengths)[0]]
        for i in range(steps):
            parts.append(layer(torch.cat([r[n + i:n + i + 1] for r, n in zip(x, lengths)]),
                               [1] * len(lengths))[0])
        full = whole(torch.cat(x), [n + steps for n in lengths])[0]
        ctx.check_device()
        # Token by token or all at once: the same attention up to the last bit's rounding.
        worst, at, before = 0, 0, 0
        for s, n in enumerate(lengths):
            rows = [parts[0][before:before + n]] + [p[s:s + 1] for p in parts[1:]]
            diff = (torch.cat(rows).int() - full[at:at + n + steps].int()).abs().max().item()
            worst, at, before = max(worst, diff), at + n + steps, before + n
        print(f"{len(lengths)} prompts of {lengths} tokens, then {steps} tokens each: "
              f"largest difference from one pass over all tokens: {worst} of 255 steps")
        return worst


if __name__ == "__main__":
    sys.exit(0 if main() <= 1 else 1)
