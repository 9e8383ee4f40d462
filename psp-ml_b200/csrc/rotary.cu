// rotary.cu - rotary positions of q and k heads, and the append of k and v
// to a paged cache.
//
// Pair (x, y) i of a head at position p turns by the angle p * f_i:
//   x' = amp * (x cos - y sin),  y' = amp * (x sin + y cos).
// f_i is held in turns per position as a 64-bit binary fraction, so p * f_i
// modulo one turn is one wrapping integer product: the angle is exact to
// 2^-64 turns per position however long the context, where a 32-bit float
// product would be off by 6e-3 rad at position 100000.  Only the reduced
// angle is rounded to a float; sums and products are 32-bit and rounded once
// to the output type.
#include <cuda_runtime.h>

#include "attention.h"

namespace pspml {

namespace {

constexpr int kThreads = 128;

template <typename In>
__device__ __forceinline__ float load1(const In* p, float scale, int32_t zero) {
  if constexpr (sizeof(In) == 1) {
    return scale * static_cast<float>(static_cast<int32_t>(*p) - zero);
  } else {
    return to_f32(*p);
  }
}

// Simple form: one element pair (or one passed-through element) per thread.
template <typename In, typename Out>
__global__ void __launch_bounds__(kThreads) k_rotary_any(const RotaryArgs a, const int units) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int64_t per_token = static_cast<int64_t>(heads) * units;
  const int64_t t = idx / per_token;
  if (t >= a.tokens) return;
  const int r = static_cast<int>(idx - t * per_token);
  int h = r / units;
  const int u = r - h * units;
  const RotaryView* w = &a.q;
  bool turned = true, cached = false;
  if (h >= a.q.heads) {
    h -= a.q.heads;
    cached = a.slots != nullptr;
    w = &a.k;
    if (h >= a.k.heads) {
      h -= a.k.heads;
      w = &a.v;
      turned = false;
    }
  }
  int64_t o = t * w->out_token;
  if (cached) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.slots_total) return;
    const int64_t page = slot / a.page_size;
    o = page * a.page_stride + (slot - page * a.page_size) * a.slot_stride;
  }
  const In* in = static_cast<const In*>(w->in) + t * w->in_token + h * w->in_head;
  Out* out = static_cast<Out*>(w->out) + o + h * w->out_head;
  const int half = a.rot / 2;
  if (u >= half) {  // passed through
    const int e = a.rot + (u - half);
    out[e] = from_f32<Out>(load1(in + e, a.scale, a.zero));
    return;
  }
  const int ex = a.layout == PSPML_ROTARY_HALF ? u : 2 * u;
  const int ey = a.layout == PSPML_ROTARY_HALF ? u + half : 2 * u + 1;
  const float x = load1(in + ex, a.scale, a.zero), y = load1(in + ey, a.scale, a.zero);
  if (!turned) {
    out[ex] = from_f32<Out>(x);
    out[ey] = from_f32<Out>(y);
    return;
  }
  const long long turns =
      static_cast<long long>(static_cast<unsigned long long>(
                                 static_cast<long long>(a.positions[t])) * a.freq[u]);
  float sn, cs;
  sincospif(static_cast<float>(turns) * 0x1p-63f, &sn, &cs);
  sn *= a.amplitude;
  cs *= a.amplitude;
  out[ex] = from_f32<Out>(x * cs - y * sn);
  out[ey] = from_f32<Out>(x * sn + y * cs);
}

template <typename In, typename Out>
cudaError_t launch_io(const RotaryArgs& a, int num_sms, cudaStream_t s) {
  (void)num_sms;
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int units = a.dim - a.rot / 2;
  const int64_t total = a.tokens * heads * units;
  const int64_t blocks = (total + kThreads - 1) / kThreads;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  k_rotary_any<In, Out><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a, units);
  return cudaGetLastError();
}

template <typename In>
cudaError_t launch_in(const RotaryArgs& a, int num_sms, cudaStream_t s) {
  switch (a.out_dtype) {
    case PSPML_DTYPE_F16: return launch_io<In, __half>(a, num_sms, s);
    case PSPML_DTYPE_BF16: return launch_io<In, __nv_bfloat16>(a, num_sms, s);
    default: return launch_io<In, float>(a, num_sms, s);
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& a, int num_sms, cudaStream_t s) {
  switch (a.in_dtype) {
    case PSPML_DTYPE_F16: return launch_in<__half>(a, num_sms, s);
    case PSPML_DTYPE_BF16: return launch_in<__nv_bfloat16>(a, num_sms, s);
    case PSPML_DTYPE_S8: return launch_in<int8_t>(a, num_sms, s);
    default: return launch_in<float>(a, num_sms, s);
  }
}

}  // namespace pspml
