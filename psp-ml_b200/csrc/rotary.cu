// rotary.cu - rotary positions of q and k heads, and the append of k and v
// to a paged cache.
//
// Pair (x, y) i of a head at position p turns by the angle p * f_i:
//   x' = amp * (x cos - y sin),  y' = amp * (x sin + y cos).
// f_i is held in turns per position as a 64-bit binary fraction, so p * f_i
// modulo one turn is one wrapping integer product, in which nothing is lost:
// the angle is as good as the frequency, a double's quotient (about 2^-53 of
// itself), times the position, 2^-24 turns for the fastest pair at position
// 2^31.  A 32-bit float product would be off by 6e-3 rad at position 100000.  Only the reduced
// angle is rounded to a float; sums and products are 32-bit and rounded once
// to the output type.
//
// Bytes bound it.  On a B200, cold: 16384 tokens of 40 F16 heads of 128, 64
// turned, 56.5 us (335 MB, 5.9 TB/s); 8191 int8 tokens of 28 + 4 + 4 heads
// appended as F16, 23.3 us (113 MB, 4.9 TB/s); 8 BF16 tokens of 40 heads 4.8 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

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

// Vector form.  The bytes bound it, so a thread moves whole vectors and
// little else: it takes V pairs of one token (elements j*V.. of both halves,
// or 2V neighbours), or V passed-through elements, and walks every
// `lanes`-th head of q, k and v with kBatch heads' loads in flight.  Blocks
// of pairs come first, then blocks of passed-through elements, so that no
// warp runs both.  Neighbouring threads take neighbouring units, then
// neighbouring heads, then tokens; a block finds the sines and cosines of
// its tokens once, in shared memory.
constexpr int kBatch = 2;

struct RotaryPlan {
  int32_t lanes;                     // heads side by side in a block
  int32_t pair_units, pass_units;    // threads a head
  int32_t pair_tokens, pass_tokens;  // tokens a block
  int64_t pair_blocks;
};

// One view's heads hl, hl + step, ... of a token.
template <typename In, typename Out, int V, bool kHalf, bool kPairs>
__device__ __forceinline__ void rotary_view(const RotaryArgs& a, const RotaryView& w, int64_t t,
                                            int64_t out_off, int hl, int step, int ex, int ey,
                                            bool turn, const float* cs, const float* sn) {
  const In* in = static_cast<const In*>(w.in) + t * w.in_token + hl * w.in_head;
  Out* out = static_cast<Out*>(w.out) + out_off + hl * w.out_head;
  const int64_t in_step = step * w.in_head, out_step = step * w.out_head;
  const float bias = 8388736.0f + static_cast<float>(a.zero);
  for (int h = hl; h < w.heads; h += kBatch * step) {
    Elems<In, V> x[kBatch], y[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (h + b * step < w.heads) {
        x[b].load(in + b * in_step + ex);
        if constexpr (kPairs) y[b].load(in + b * in_step + ey);
      }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (h + b * step < w.heads) {
        Elems<Out, V> o;
        if constexpr (!kPairs && std::is_same<In, Out>::value) {
          x[b].store(out + b * out_step + ex);
        } else if constexpr (!kPairs) {
          float v[V];
          x[b].values(v, a.scale, bias);
          o.round(v);
          o.store(out + b * out_step + ex);
        } else {
          float v[2 * V];
          x[b].values(v, a.scale, bias);
          y[b].values(v + V, a.scale, bias);
          if (turn) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float& p = kHalf ? v[i] : v[2 * i];
              float& q = kHalf ? v[V + i] : v[2 * i + 1];
              const float s = p * cs[i] - q * sn[i];
              q = p * sn[i] + q * cs[i];
              p = s;
            }
          }
          o.round(v);
          o.store(out + b * out_step + ex);
          o.round(v + V);
          o.store(out + b * out_step + ey);
        }
      }
    in += kBatch * in_step;
    out += kBatch * out_step;
  }
}

template <typename In, typename Out, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads, 8)
    k_rotary_vec(const RotaryArgs a, const RotaryPlan pl) {
  __shared__ float2 s_turn[kThreads * V];  // [token][pair]: pair_tokens * pair_units <= kThreads
  const bool pairs = blockIdx.x < pl.pair_blocks;
  const int units = pairs ? pl.pair_units : pl.pass_units;
  const int tokens = pairs ? pl.pair_tokens : pl.pass_tokens;
  const int64_t t0 = (pairs ? static_cast<int64_t>(blockIdx.x)
                            : static_cast<int64_t>(blockIdx.x) - pl.pair_blocks) * tokens;
  const int tl = threadIdx.x / (units * pl.lanes);
  const int rest = threadIdx.x - tl * (units * pl.lanes);
  const int u = rest % units;
  const int hl = blockIdx.y * pl.lanes + rest / units, step = gridDim.y * pl.lanes;
  const int64_t t = t0 + tl;
  const int half = a.rot / 2;

  if (pairs) {
    for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
      const int64_t ti = t0 + i / half;
      if (ti < a.tokens) {
        const unsigned long long at =
            static_cast<unsigned long long>(static_cast<long long>(a.positions[ti]));
        float sn, cs;
        sincospif(static_cast<float>(static_cast<long long>(at * a.freq[i % half])) * 0x1p-63f, &sn,
                  &cs);
        s_turn[i] = make_float2(cs * a.amplitude, sn * a.amplitude);
      }
    }
    __syncthreads();
  }
  if (tl >= tokens || t >= a.tokens) return;

  int64_t cached = 0;  // offset of the token's slot
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
  const int64_t k_off = a.slots != nullptr ? cached : t * a.k.out_token;
  if (pairs) {
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 c = s_turn[tl * half + u * V + i];
      cs[i] = c.x;
      sn[i] = c.y;
    }
    const int ex = kHalf ? u * V : u * 2 * V, ey = kHalf ? ex + half : ex + V;
    rotary_view<In, Out, V, kHalf, true>(a, a.q, t, t * a.q.out_token, hl, step, ex, ey, true, cs,
                                         sn);
    if (!keep) return;
    rotary_view<In, Out, V, kHalf, true>(a, a.k, t, k_off, hl, step, ex, ey, true, cs, sn);
    rotary_view<In, Out, V, kHalf, true>(a, a.v, t, cached, hl, step, ex, ey, false, cs, sn);
  } else {
    const int e = a.rot + u * V;
    rotary_view<In, Out, V, kHalf, false>(a, a.q, t, t * a.q.out_token, hl, step, e, 0, false,
                                          nullptr, nullptr);
    if (!keep) return;
    rotary_view<In, Out, V, kHalf, false>(a, a.k, t, k_off, hl, step, e, 0, false, nullptr, nullptr);
    rotary_view<In, Out, V, kHalf, false>(a, a.v, t, cached, hl, step, e, 0, false, nullptr, nullptr);
  }
}

// Whether every vector of V elements is aligned in memory.
template <typename In, typename Out, int V>
bool vectors_fit(const RotaryArgs& a) {
  if (a.rot % (2 * V) != 0 || a.dim % V != 0 || a.rot / (2 * V) > kThreads ||
      (a.dim - a.rot) / V > kThreads)
    return false;
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
  const int heads = std::max({a.q.heads, a.k.heads, a.v.heads});
  RotaryPlan pl{};
  pl.pair_units = a.rot / (2 * V);
  pl.pass_units = (a.dim - a.rot) / V;
  const int units = pl.pair_units + pl.pass_units, most = std::max(pl.pair_units, pl.pass_units);
  // Four heads side by side when tokens are many: long runs in memory, and
  // a thread uses its angles for a quarter of the heads.  With few tokens
  // the heads are spread over blocks until the machine is full of threads.
  pl.lanes = std::max(1, std::min({4, heads, kThreads / most}));
  int split = 1;
  while (split * pl.lanes < heads && split < 32768 &&
         a.tokens * units * pl.lanes * split < static_cast<int64_t>(num_sms) * 1024)
    split *= 2;
  int64_t blocks = 0;
  if (pl.pair_units > 0) {
    pl.pair_tokens = kThreads / (pl.pair_units * pl.lanes);
    pl.pair_blocks = (a.tokens + pl.pair_tokens - 1) / pl.pair_tokens;
    blocks += pl.pair_blocks;
  }
  if (pl.pass_units > 0) {
    pl.pass_tokens = kThreads / (pl.pass_units * pl.lanes);
    blocks += (a.tokens + pl.pass_tokens - 1) / pl.pass_tokens;
  }
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(split));
  if (a.layout == PSPML_ROTARY_HALF)
    k_rotary_vec<In, Out, V, true><<<grid, kThreads, 0, s>>>(a, pl);
  else
    k_rotary_vec<In, Out, V, false><<<grid, kThreads, 0, s>>>(a, pl);
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
