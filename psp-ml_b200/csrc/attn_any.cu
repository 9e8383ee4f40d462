// attn_any.cu - attention on CUDA cores for any type, head size, stride and
// alignment.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale * q_i.k_j - m_i)
// over the keys j that row i's masks leave, in one pass over the keys: a
// block takes one row of one head, each of its warps every fourth 32 keys
// with a running maximum m and sum, one key per lane for the products q.k
// and the head's elements spread over the lanes for the sums of v.  Masked
// keys are never read, so nothing they hold can reach a row.  Products,
// statistics and sums are 32-bit; only the output is rounded.
//
// Latency bounds it (a lane's product of a whole head, uncoalesced): it is
// here for coverage.  On a B200 one token over 777 keys of 8/2 heads of 64
// takes 82 us, a prompt of 37 such tokens 16 us.
#include <cuda_runtime.h>

#include <cmath>

#include "attention.h"

namespace pspml {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxDim = 256;
constexpr int kPerLane = kMaxDim / 32;

// Element offset of key j's row in the pools, or -1 for a page outside them.
__device__ __forceinline__ int64_t paged_row(const AttnArgs& a, const int32_t* table, int64_t j) {
  const int64_t i = j / a.page_size;
  const int64_t page = table[i];
  if (page < 0 || page >= a.n_pages) return -1;
  return page * a.page_stride + (j - i * a.page_size) * a.kv_token;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) k_attn_any(const AttnArgs a) {
  const int64_t row = blockIdx.x / a.q_heads;
  const int head = static_cast<int>(blockIdx.x - row * a.q_heads);
  __shared__ float sq[kMaxDim];
  __shared__ float so[kWarps][kMaxDim];
  __shared__ float sm[kWarps], sl[kWarps];

  // The sequence that holds the row: the last one starting at or before it.
  int lo = 0, hi = a.sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= row) lo = mid; else hi = mid;
  }
  const SeqSpan sp = seq_span(a, lo);
  const int64_t r = row - sp.begin;
  if (r < 0 || r >= sp.rows || (a.paged && r >= a.max_new)) return;

  const T* q = static_cast<const T*>(a.q) + row * a.q_token + head * a.q_head;
  for (int e = threadIdx.x; e < a.dim; e += kWarps * 32) sq[e] = to_f32(q[e]);
  __syncthreads();

  const int kvh = head / (a.q_heads / a.kv_heads);
  const int64_t place = sp.keys - sp.rows + r;
  int64_t end = sp.keys, begin = 0;
  if (a.causal && place + 1 < end) end = place + 1;
  if (a.window > 0 && place - a.window + 1 > 0) begin = place - a.window + 1;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int32_t* table = a.paged ? a.pages + lo * a.pages_stride : nullptr;
  const T* kb = static_cast<const T*>(a.k) + kvh * a.kv_head;
  const T* vb = static_cast<const T*>(a.v) + kvh * a.v_head;
  float m = -INFINITY, l = 0.0f, acc[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) acc[i] = 0.0f;

  for (int64_t j0 = begin + warp * 32; j0 < end; j0 += kWarps * 32) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    int64_t vrow = -1;
    if (j < end) {
      const int64_t krow = a.paged ? paged_row(a, table, j) : (sp.begin + j) * a.kv_token;
      vrow = a.paged ? krow : (sp.begin + j) * a.v_token;
      float dot = 0.0f;
      if (krow >= 0)
        for (int e = 0; e < a.dim; ++e) dot = fmaf(sq[e], to_f32(kb[krow + e]), dot);
      s = dot * a.scale;
    }
    float top = s;
#pragma unroll
    for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float m2 = fmaxf(m, top);
    // -inf only while every score so far is -inf (an infinite product).
    const float base = m2 == -INFINITY ? 0.0f : m2;
    const float p = j < end ? expf(s - base) : 0.0f;
    const float fix = expf(m - base);
    m = m2;
    l = l * fix + p;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) acc[i] *= fix;
    const int n = static_cast<int>(end - j0 < 32 ? end - j0 : 32);
    for (int x = 0; x < n; ++x) {
      const float px = __shfl_sync(~0u, p, x);
      const int64_t vx = __shfl_sync(~0u, vrow, x);
      if (vx < 0) continue;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (lane + 32 * i < a.dim) acc[i] = fmaf(px, to_f32(vb[vx + lane + 32 * i]), acc[i]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) l += __shfl_xor_sync(~0u, l, o);
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) so[warp][lane + 32 * i] = acc[i];
  __syncthreads();

  float top = sm[0];
  for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, f[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    f[w] = expf(sm[w] - base);
    sum += sl[w] * f[w];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int e = threadIdx.x; e < a.dim; e += kWarps * 32) {
    float o = 0.0f;
    for (int w = 0; w < kWarps; ++w) o += so[w][e] * f[w];
    o *= inv;
    const int64_t at = row * a.o_token + head * a.o_head + e;
    if (a.out_dtype == PSPML_DTYPE_S8)
      static_cast<int8_t*>(a.out)[at] = quantise_s8(o, a.out_inv_scale, a.out_zero);
    else
      static_cast<T*>(a.out)[at] = from_f32<T>(o);
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[row * a.q_heads + head] = sum == 0.0f ? -INFINITY : logf(sum) + base;
}

}  // namespace

cudaError_t launch_attn_any(const AttnArgs& a, cudaStream_t s) {
  const int64_t blocks = a.tokens * a.q_heads;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(blocks);
  switch (a.dtype) {
    case PSPML_DTYPE_F16: k_attn_any<__half><<<grid, kWarps * 32, 0, s>>>(a); break;
    case PSPML_DTYPE_BF16: k_attn_any<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(a); break;
    default: k_attn_any<float><<<grid, kWarps * 32, 0, s>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace pspml
