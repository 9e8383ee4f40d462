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

#include <algorithm>

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

// V neighbouring elements, moved in pieces of at most 16 bytes.
template <int Bytes> struct Piece;
template <> struct Piece<4> { using type = uint32_t; };
template <> struct Piece<8> { using type = uint2; };
template <> struct Piece<16> { using type = uint4; };
template <typename E, int V>
struct Elems {
  static constexpr int kPiece = V * sizeof(E) < 16 ? V * sizeof(E) : 16;
  static constexpr int kPieces = V * sizeof(E) / kPiece;
  using P = typename Piece<kPiece>::type;
  P p[kPieces];
  __device__ __forceinline__ void load(const E* s) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) p[i] = reinterpret_cast<const P*>(s)[i];
  }
  __device__ __forceinline__ void store(E* d) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<P*>(d)[i] = p[i];
  }
  __device__ __forceinline__ uint32_t& word(int i) { return reinterpret_cast<uint32_t*>(p)[i]; }
  // Values as floats; `bias` is 2^23 + 128 + zero point for S8.
  __device__ __forceinline__ void values(float* v, float scale, float bias) {
    if constexpr (sizeof(E) == 1) {
      // A byte with its sign bit flipped is q + 128; as the low byte of the
      // float 2^23 it adds to it exactly, with no conversion instruction.
#pragma unroll
      for (int i = 0; i < V; ++i)
        v[i] = scale * (__uint_as_float(__byte_perm(word(i / 4) ^ 0x80808080u, 0x4B000000u,
                                                    0x7540 + (i % 4))) - bias);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = to_f32(reinterpret_cast<const E*>(p)[i]);
    }
  }
  __device__ __forceinline__ void round(const float* v) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) word(i) = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) word(i) = pack2<E>(v[2 * i], v[2 * i + 1]);
    }
  }
};

// Vector form.  The bytes bound it, so a thread moves whole vectors: it
// takes V pairs of one token (elements j*V.. of both halves, or 2V
// neighbours) or V passed-through elements, finds their sines and cosines
// once, and walks every `lanes`-th head with kBatch heads' loads in flight.
// Neighbouring threads take neighbouring units, then neighbouring heads, so
// a step of a warp covers whole heads side by side in memory.
constexpr int kBatch = 4;
template <typename In, typename Out, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads)
    k_rotary_vec(const RotaryArgs a, const int units, const int lanes) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t t = idx / (units * lanes);
  if (t >= a.tokens) return;
  const int rest = static_cast<int>(idx - t * (units * lanes));
  const int hl = rest / units, u = rest - hl * units;
  const int turned = a.rot / (2 * V);      // units that hold pairs
  const bool pairs = u < turned;
  const int ex = pairs ? (kHalf ? u * V : u * 2 * V) : a.rot + (u - turned) * V;
  const int ey = kHalf ? ex + a.rot / 2 : ex + V;
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const float bias = 8388736.0f + static_cast<float>(a.zero);

  int64_t cached = 0;                       // offset of the token's slot
  bool keep = true;
  if (a.slots != nullptr) {
    const int64_t slot = a.slots[t];
    keep = slot >= 0 && slot < a.slots_total;
    if (keep) {
      const int64_t page = (slot >> 32) == 0 ? static_cast<uint32_t>(slot) /
                                                   static_cast<uint32_t>(a.page_size)
                                             : slot / a.page_size;
      cached = page * a.page_stride + (slot - page * a.page_size) * a.slot_stride;
    }
  }
  float sn[V], cs[V];
  if (pairs) {
    const unsigned long long at =
        static_cast<unsigned long long>(static_cast<long long>(a.positions[t]));
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const long long turns = static_cast<long long>(at * a.freq[u * V + i]);
      sincospif(static_cast<float>(turns) * 0x1p-63f, &sn[i], &cs[i]);
      sn[i] *= a.amplitude;
      cs[i] *= a.amplitude;
    }
  }

  for (int hb = hl; hb < heads; hb += kBatch * lanes) {
    Elems<In, V> x[kBatch], y[kBatch];
    Out* dst[kBatch];
    bool turn[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      int h = hb + b * lanes;
      dst[b] = nullptr;
      if (h >= heads) continue;
      const bool is_q = h < a.q.heads;
      if (!is_q) h -= a.q.heads;
      const bool is_k = !is_q && h < a.k.heads;
      if (!is_q && !is_k) h -= a.k.heads;
      turn[b] = is_q || is_k;
      const RotaryView& w = is_q ? a.q : (is_k ? a.k : a.v);
      const bool to_cache = !is_q && a.slots != nullptr;
      if (to_cache && !keep) continue;
      dst[b] = static_cast<Out*>(w.out) + (to_cache ? cached : t * w.out_token) + h * w.out_head;
      const In* src = static_cast<const In*>(w.in) + t * w.in_token + h * w.in_head;
      x[b].load(src + ex);
      if (pairs) y[b].load(src + ey);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (dst[b] == nullptr) continue;
      float v[2 * V];
      x[b].values(v, a.scale, bias);
      if (pairs) y[b].values(v + V, a.scale, bias);
      if (pairs && turn[b]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float& p = kHalf ? v[i] : v[2 * i];
          float& q = kHalf ? v[V + i] : v[2 * i + 1];
          const float s = p * cs[i] - q * sn[i];
          q = p * sn[i] + q * cs[i];
          p = s;
        }
      }
      Elems<Out, V> o;
      o.round(v);
      o.store(dst[b] + ex);
      if (pairs) {
        o.round(v + V);
        o.store(dst[b] + ey);
      }
    }
  }
}

// Whether every vector of V elements is aligned in memory.
template <typename In, typename Out, int V>
bool vectors_fit(const RotaryArgs& a) {
  if (a.rot % (2 * V) != 0 || a.dim % V != 0) return false;
  const auto fits = [](const void* p, int64_t bits, int bytes) {
    const int n = bytes < 16 ? bytes : 16;
    return reinterpret_cast<uintptr_t>(p) % n == 0 && (bits * (bytes / V)) % n == 0;
  };
  const int in = V * sizeof(In), out = V * sizeof(Out);
  for (const RotaryView* w : {&a.q, &a.k, &a.v}) {
    if (w->heads == 0) continue;
    if (!fits(w->in, w->in_token | w->in_head, in) || !fits(w->out, w->out_token | w->out_head, out))
      return false;
  }
  return a.slots == nullptr || fits(nullptr, a.page_stride | a.slot_stride, out);
}

template <typename In, typename Out, int V>
cudaError_t launch_vec(const RotaryArgs& a, int num_sms, cudaStream_t s) {
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int units = a.dim / V - a.rot / (2 * V);
  // Threads a token and unit: four when tokens are many, so that a thread
  // uses its angles for a quarter of the heads; more until the machine is
  // full of threads, up to one a head.
  int lanes = std::min(4, heads);
  while (lanes < heads && a.tokens * units * lanes < static_cast<int64_t>(num_sms) * 1024)
    lanes = std::min(2 * lanes, heads);
  const int64_t blocks = (a.tokens * units * lanes + kThreads - 1) / kThreads;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (a.layout == PSPML_ROTARY_HALF)
    k_rotary_vec<In, Out, V, true><<<grid, kThreads, 0, s>>>(a, units, lanes);
  else
    k_rotary_vec<In, Out, V, false><<<grid, kThreads, 0, s>>>(a, units, lanes);
  return cudaGetLastError();
}

template <typename In, typename Out>
cudaError_t launch_io(const RotaryArgs& a, int num_sms, cudaStream_t s) {
  // Eight elements where 16-byte vectors of them fit, four where half-size
  // ones do (a rotated part that is no multiple of 16).
  if constexpr (sizeof(In) <= 2 && sizeof(Out) <= 2)
    if (vectors_fit<In, Out, 8>(a)) return launch_vec<In, Out, 8>(a, num_sms, s);
  if (vectors_fit<In, Out, 4>(a)) return launch_vec<In, Out, 4>(a, num_sms, s);
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
