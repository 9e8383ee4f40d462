// attention.h - launches of the attention operators (host C++).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/pspml.h"
#include "runtime.h"

// Keeps what it needs of its context, so that it may be used and destroyed
// after it.
struct pspml_rotary {
  int device = 0;
  int num_sms = 0;
  pspml_rotary_desc d{};
  unsigned long long* freq = nullptr;  // device: rot_dim/2 turns per position, 64-bit fractions
};

namespace pspml {

// Arguments of both attention calls, checked.  `paged`: keys and values
// come from the cache (kv_* then hold its strides), else they are packed
// like q.
struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
  const int32_t* starts;
  const int32_t* lengths;
  const int32_t* pages;
  int64_t tokens;
  int64_t q_token, q_head;      // strides, elements
  int64_t kv_token, kv_head;    // k: packed token stride, or slot stride of a page
  int64_t v_token, v_head;
  int64_t page_stride, pages_stride, n_pages;
  int64_t o_token, o_head;
  int32_t sequences, q_heads, kv_heads, dim, page_size, max_new;
  int32_t causal, window, paged;
  int32_t dtype, out_dtype;
  float scale;
  float out_inv_scale;          // S8 output: round(o * out_inv_scale) + out_zero
  int32_t out_zero;
};

// One sequence of a call, with every index clamped to the call's buffers.
struct SeqSpan {
  int64_t begin;   // first row in q
  int64_t keys;
  int64_t rows;
};
__device__ __forceinline__ SeqSpan seq_span(const AttnArgs& a, int s) {
  SeqSpan r;
  const int64_t b = a.starts[s], e = a.starts[s + 1];
  r.begin = b < 0 ? 0 : (b > a.tokens ? a.tokens : b);
  const int64_t end = e < r.begin ? r.begin : (e > a.tokens ? a.tokens : e);
  r.rows = end - r.begin;
  if (a.paged) {
    const int64_t n = a.lengths[s], most = a.pages_stride * a.page_size;
    r.keys = n < 0 ? 0 : (n > most ? most : n);
  } else {
    r.keys = r.rows;
  }
  return r;
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
// Two values rounded into one 32-bit word, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^x as the special function unit gives it (2^-22 relative).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The int8 an output value is stored as: nearest (ties to even), clamped
// while still a float so that infinities saturate; NaN gives the zero point.
__device__ __forceinline__ int8_t quantise_s8(float v, float inv_scale, int32_t zero) {
  const float r = rintf(v * inv_scale) + static_cast<float>(zero);
  return static_cast<int8_t>(
      r != r ? zero : static_cast<int32_t>(fminf(fmaxf(r, -128.0f), 127.0f)));
}

struct RotaryView {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;
  int32_t heads;
};
struct RotaryArgs {
  RotaryView q, k, v;  // heads 0: absent
  const int32_t* positions;
  const int64_t* slots;       // NULL: k goes to a plain view
  const unsigned long long* freq;
  int64_t page_stride, slot_stride, slots_total;  // cache
  int64_t tokens;
  int32_t page_size, dim, rot, layout;
  int32_t in_dtype, out_dtype, zero;
  float scale, amplitude;
};

// What a split call may use between its CTAs.
struct AttnWork {
  uint8_t* base;        // attn_workspace_bytes(num_sms)
  unsigned* counters;   // kAttnCounters words, zero between calls
  unsigned* err;        // the context's device error word
  int num_sms;
};

cudaError_t launch_rotary(const RotaryArgs& a, int num_sms, cudaStream_t s);
// Two pieces a CTA, one CTA an SM, of 256 rows of 128 sums, a maximum and a
// sum (attn_tc.cu; the 16-row pieces of attn_step.cu need less).
inline size_t attn_workspace_bytes(int num_sms) {
  return static_cast<size_t>(2 * num_sms) * 256 * (128 * sizeof(float) + sizeof(float2));
}

cudaError_t launch_attn_any(const AttnArgs& a, cudaStream_t s);
cudaError_t launch_attn_step(const AttnArgs& a, const AttnWork& w, cudaStream_t s);
bool attn_tc_covers(const AttnArgs& a);
cudaError_t launch_attn_tc(const AttnArgs& a, const AttnWork& w, cudaStream_t s);

}  // namespace pspml
