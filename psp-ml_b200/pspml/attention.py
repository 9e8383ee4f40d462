"""Rotary positions, the paged key/value cache and attention on torch tensors.

A thin mirror of the attention section of include/pspml.h: each function
describes its tensors to the C ABI and makes one call.  Heads are tensors
[tokens][heads][dim] whose last dimension is contiguous (slices of one
projection's output are fine); index tensors are contiguous.  Everything is
asynchronous on `stream` (a cudaStream_t as an int; 0 is the legacy default
stream, and without one it is torch's current stream), nothing is kept from one call to the next, and errors raise
PspmlError.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np
import torch

from . import capi

_ref = ctypes.byref
_DTYPES = {torch.float32: capi.DTYPE_F32, torch.float16: capi.DTYPE_F16,
           torch.bfloat16: capi.DTYPE_BF16}
_LAYOUTS = {"half": capi.ROTARY_HALF, "interleaved": capi.ROTARY_INTERLEAVED}
_SCALINGS = {"none": capi.ROTARY_SCALE_NONE, "linear": capi.ROTARY_SCALE_LINEAR,
             "base": capi.ROTARY_SCALE_BASE, "parts": capi.ROTARY_SCALE_PARTS}


class Quantised:
    """int8 heads standing for scale * (tensor - zero_point)."""

    def __init__(self, tensor: torch.Tensor, scale: float, zero_point: int = 0):
        if tensor.dtype != torch.int8:
            raise ValueError("Quantised takes an int8 tensor")
        self.tensor, self.scale, self.zero_point = tensor, scale, zero_point


def _on(device: int, t: torch.Tensor, what: str) -> None:
    if t.get_device() != device:
        raise ValueError(f"{what} is on {t.device}, the context on cuda:{device}")


# struct pspml_heads and pspml_attention_desc as bytes: half the cost of filling a
# ctypes.Structure.
_pack_heads = struct.Struct("@Pqqiiiifi").pack
_pack_desc = struct.Struct("@fiii").pack


def heads(x, device: int, what: str = "tensor", tokens: int | None = None) -> bytes:
    """The C view (struct pspml_heads) of a [tokens][heads][dim] tensor or a Quantised one."""
    if type(x) is Quantised:
        x, scale, zero, dtype = x.tensor, x.scale, x.zero_point, capi.DTYPE_S8
    else:
        scale, zero, dtype = 1.0, 0, _DTYPES.get(x.dtype)
        if dtype is None:
            raise ValueError(f"{what}: dtype {x.dtype} is not float32, float16 or bfloat16")
    if x.get_device() != device:
        _on(device, x, what)
    n, h, d = x.shape
    if tokens is not None and n != tokens:
        raise ValueError(f"{what}: {n} tokens in a call of {tokens}")
    st, sh, sd = x.stride()
    if sd != 1 and d != 1:
        raise ValueError(f"{what}: a head's elements are not contiguous")
    return _pack_heads(x.data_ptr(), st, sh, h, d, dtype, zero, scale, 0)


def _index(x: torch.Tensor, dtype, n: int, device: int, what: str) -> int:
    if x.dtype is not dtype or x.numel() != n or not x.is_contiguous():
        raise ValueError(f"{what}: needs {n} contiguous {dtype}")
    if x.get_device() != device:
        _on(device, x, what)
    return x.data_ptr()


def _stream(stream: int | None, device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream if stream is None else stream


class Rotary:
    """Rotary positions of one head shape (pspml_rotary).

    layout "half" pairs element i with i + rot_dim/2, "interleaved" 2i with
    2i + 1; scaling "none", "linear", "base" or "parts" (see pspml.h)."""

    def __init__(self, ctx: capi.Context, head_dim: int, rot_dim: int | None = None,
                 layout: str = "half", base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, original_len: float = 0.0, low: float = 1.0,
                 high: float = 4.0, amplitude: float = 1.0):
        self.ctx = ctx
        self.desc = rotary_desc(head_dim, rot_dim, layout, base, scaling, factor, original_len,
                                low, high, amplitude)
        self.handle = ctypes.c_void_p()
        capi.call("pspml_rotary_create", ctx.handle, _ref(self.desc),
                  _ref(self.handle))

    def close(self) -> None:
        if self.handle:
            self.ctx.lib.pspml_rotary_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def rotary_desc(head_dim, rot_dim=None, layout="half", base=10000.0, scaling="none", factor=1.0,
                original_len=0.0, low=1.0, high=4.0, amplitude=1.0) -> capi.RotaryDesc:
    return capi.RotaryDesc(head_dim, head_dim if rot_dim is None else rot_dim, _LAYOUTS[layout],
                           _SCALINGS[scaling], base, factor, low, high, original_len, amplitude)


def rotary_frequencies(desc: capi.RotaryDesc) -> np.ndarray:
    """Turns per position of each pair, as 64-bit binary fractions of a turn (no device)."""
    out = np.zeros(max(1, desc.rot_dim // 2), np.uint64)
    capi.call("pspml_rotary_frequencies", _ref(desc), out.ctypes.data)
    return out[:desc.rot_dim // 2]


class KvCache:
    """Paged key and value pools, tensors [pages][page_size][heads][dim] of equal strides whose
    last dimension is contiguous (a transposed [pages][heads][page_size][dim] tensor is fine)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise ValueError("key and value pools differ in shape, strides or dtype")
        if k.dim() != 4 or (k.stride(3) != 1 and k.shape[3] != 1):
            raise ValueError("a pool is [pages][page_size][heads][dim], the last contiguous")
        if k.dtype not in _DTYPES:
            raise ValueError(f"pool dtype {k.dtype} is not float32, float16 or bfloat16")
        if k.device != v.device:
            raise ValueError("key and value pools are on different devices")
        self.k, self.v = k, v
        pages, size, n, d = k.shape
        sp, ss, sh, _ = k.stride()
        self.view = capi.KvCacheView(k.data_ptr(), v.data_ptr(), sp, ss, sh, pages, size, n, d,
                                     _DTYPES[k.dtype])


def _tokens(x) -> int:
    return (x.tensor if type(x) is Quantised else x).shape[0]


def rotary_apply(rotary: Rotary, positions: torch.Tensor, q, q_out, k=None, k_out=None,
                 stream: int | None = None) -> None:
    """q_out, k_out = q, k turned to their int32 positions; outputs may be the inputs."""
    n, dev = _tokens(q), rotary.ctx.device
    status = rotary.ctx.lib.pspml_rotary_apply(
        rotary.handle, n, _index(positions, torch.int32, n, dev, "positions"),
        heads(q, dev, "q"), heads(q_out, dev, "q_out", n),
        heads(k, dev, "k", n) if k is not None else None,
        heads(k_out, dev, "k_out", n) if k_out is not None else None, _stream(stream, dev))
    if status:
        capi.check(status, "pspml_rotary_apply")


def rotary_append(rotary: Rotary, positions: torch.Tensor, slots: torch.Tensor, q, q_out, k, v,
                  cache: KvCache, stream: int | None = None) -> None:
    """q_out = q turned to its positions (q and q_out may be None); token t's turned k and its v
    go to slot slots[t] = page * page_size + slot of the cache (int64; outside it: skipped)."""
    n, dev = _tokens(k), rotary.ctx.device
    _on(dev, cache.k, "cache")
    status = rotary.ctx.lib.pspml_rotary_append(
        rotary.handle, n, _index(positions, torch.int32, n, dev, "positions"),
        _index(slots, torch.int64, n, dev, "slots"),
        heads(q, dev, "q", n) if q is not None else None,
        heads(q_out, dev, "q_out", n) if q_out is not None else None,
        heads(k, dev, "k"), heads(v, dev, "v", n), _ref(cache.view), _stream(stream, dev))
    if status:
        capi.check(status, "pspml_rotary_append")


def _desc(dim: int, causal: bool, window: int, scale: float | None) -> bytes:
    return _pack_desc(dim ** -0.5 if scale is None else scale, 1 if causal else 0, window, 0)


def _lse(lse, q, dev) -> int:
    return _index(lse, torch.float32, q.shape[0] * q.shape[1], dev, "lse")


def prompt(ctx: capi.Context, q, k, v, starts: torch.Tensor, out, lse=None, causal: bool = True,
           window: int = 0, scale: float | None = None, stream: int | None = None) -> None:
    """Attention over packed whole prompts: sequence s is tokens starts[s] .. starts[s+1] (int32)
    of q, k, v and out; scale defaults to dim ** -0.5; lse [tokens][heads] float32 or None."""
    dev = ctx.device
    n, _, dim = q.shape
    edges = starts.numel()
    status = ctx.lib.pspml_attention_prompt(
        ctx.handle, _desc(dim, causal, window, scale), n, edges - 1,
        _index(starts, torch.int32, edges, dev, "starts"), heads(q, dev, "q"),
        heads(k, dev, "k", n), heads(v, dev, "v", n), heads(out, dev, "out", n),
        None if lse is None else _lse(lse, q, dev), _stream(stream, dev))
    if status:
        capi.check(status, "pspml_attention_prompt")


def cached(ctx: capi.Context, q, cache: KvCache, starts: torch.Tensor, lengths: torch.Tensor,
           pages: torch.Tensor, out, max_new: int, lse=None, causal: bool = True, window: int = 0,
           scale: float | None = None, stream: int | None = None) -> None:
    """Attention of each sequence's new tokens starts[s] .. starts[s+1] of q, at most max_new,
    over its lengths[s] cached keys (the new ones among them), found through row s of the int32
    page table `pages`."""
    dev = ctx.device
    n, _, dim = q.shape
    seqs = starts.numel() - 1
    _on(dev, cache.k, "cache")
    _on(dev, pages, "pages")
    if pages.dtype is not torch.int32 or pages.dim() != 2 or not pages.is_contiguous() or \
            pages.shape[0] != seqs:
        raise ValueError("pages: needs a contiguous int32 row for each sequence")
    status = ctx.lib.pspml_attention_cached(
        ctx.handle, _desc(dim, causal, window, scale), n, seqs, max_new,
        _index(starts, torch.int32, seqs + 1, dev, "starts"),
        _index(lengths, torch.int32, seqs, dev, "lengths"), pages.data_ptr(), pages.shape[1],
        heads(q, dev, "q"), _ref(cache.view), heads(out, dev, "out", n),
        None if lse is None else _lse(lse, q, dev), _stream(stream, dev))
    if status:
        capi.check(status, "pspml_attention_cached")
