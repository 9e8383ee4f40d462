// attn_rows.cuh - rows of a tile again, by a warp, without their masked keys.
//
// A tile's product P V multiplies the keys that a row's mask leaves out by a
// weight of 0.  Where such a key's values are not finite, 0 * v is NaN and
// the row is lost although it does not see the key.  The tile kernels look at
// their outputs (a multiply-add a value) and come here with the rows that are
// not finite:
//   1. a token's rows are done again only if a masked key among those that
//      were multiplied has a non-finite value in a column that the keys the
//      token sees have not settled.  A NaN among them settles a column, and so
//      do infinities of both signs: whatever the weights, the sum is NaN with
//      and without the masked keys.  One sign alone does not: the formula
//      gives that infinity, 0 * v turned it into NaN;
//   2. eight rows at a time: a lane holds a few columns of all eight, and each
//      key is read once; a row's score is summed over the lanes and kept by
//      four of them, and values of keys that a row does not see are skipped.
// Infinities that a row does see count with the weight that the tile used: one
// that rounds to 0 in the operands' type (below 2^-25 in F16) makes NaN of them.
// Finite outputs never come here.  One bad token costs the rows of the tokens
// that share its tile one more pass over their keys, at most 127 tokens' of a
// prompt, bound by latency on few warps: 16384 tokens of 32 heads take 51 ms
// with token 12127 bad, 3 ms with token 100 or all of them NaN, 0.5 s with an
// infinity in one column of all of them (no row is settled), 1.7 ms with none
// bad.  Sums and statistics are 32-bit, weights are not rounded.
#pragma once

#include <cmath>

#include "attention.h"

namespace pspml {

// Rows of one sequence and key head: row i is token i / group of the head
// i % group of the group.
struct AttnRows {
  const int32_t* table;  // pages of the sequence, paged only
  int64_t begin;         // the sequence's first row in packed keys
  int64_t keys;          // of the sequence
  int64_t lo, hi;        // keys that were multiplied
  int64_t row0, place0;  // row in q and out, and position, of row 0's token
  int32_t head, group;
  int32_t first;         // row of bit 0 of the mask
};

template <typename T, int C>
struct alignas(C * sizeof(T)) AttnColumns {
  T x[C];
};

template <typename T, int DP>
__device__ __noinline__ void attn_rows_again(const AttnArgs& a, const AttnRows& r, uint32_t bad) {
  constexpr int C = DP / 32, kGroup = 8, kBatch = 4, kScan = 8;
  using Columns = AttnColumns<T, C>;
  const int lane = threadIdx.x % 32, e0 = lane * C;
  const bool live = e0 < a.dim;
  const T* const kb = static_cast<const T*>(a.k) + r.head * a.kv_head + e0;
  const T* const vb = static_cast<const T*>(a.v) + r.head * a.v_head + e0;

  // Where key j's keys and values start; false for a page outside the pools.
  const int64_t k_stride = a.kv_token, v_stride = a.v_token, page_stride = a.page_stride;
  const int64_t packed = r.begin, n_pages = a.n_pages;
  const uint32_t page_size = a.page_size;
  const int32_t* const table = r.table;
  auto key_at = [&](int64_t j, int64_t* k, int64_t* v) {
    if (table == nullptr) {
      *k = (packed + j) * k_stride;
      *v = (packed + j) * v_stride;
      return true;
    }
    const uint32_t i = static_cast<uint32_t>(j) / page_size;
    const int64_t page = table[i];
    *k = *v = page * page_stride + (static_cast<uint32_t>(j) - i * page_size) * k_stride;
    return page >= 0 && page < n_pages;
  };
  auto load = [&](const T* base, int64_t at, bool real) {
    Columns c;
    if (real) {
      c = *reinterpret_cast<const Columns*>(base + at);
    } else {
#pragma unroll
      for (int x = 0; x < C; ++x) c.x[x] = from_f32<T>(0.0f);
    }
    return c;
  };
  auto end_of = [&](int64_t place) {
    return a.causal && place + 1 < r.keys ? place + 1 : r.keys;
  };
  auto begin_of = [&](int64_t place) {
    return a.window > 0 && place - a.window + 1 > 0 ? place - a.window + 1 : int64_t{0};
  };
  // The lane's columns in which keys of [j0, j1) hold a value that is not
  // finite (`seen` false), or values that make any weighted sum NaN (`seen`
  // true); over once all columns of `stop` have been found.
  auto bad_columns = [&](int64_t j0, int64_t j1, bool seen, uint32_t stop) {
    uint32_t nan = 0, above = 0, below = 0, found = 0;
    for (int64_t j = j1; j > j0; j -= kScan) {
      Columns c[kScan];
#pragma unroll
      for (int b = 0; b < kScan; ++b) {
        int64_t k, v;
        const bool real = j - 1 - b >= j0 && key_at(j - 1 - b, &k, &v);
        c[b] = load(vb, v, real && live);
      }
#pragma unroll
      for (int b = 0; b < kScan; ++b)
#pragma unroll
        for (int x = 0; x < C; ++x) {
          const float f = to_f32(c[b].x[x]);
          nan |= f != f ? 1u << x : 0u;
          above |= f == INFINITY ? 1u << x : 0u;
          below |= f == -INFINITY ? 1u << x : 0u;
        }
      found = nan | (seen ? above & below : above | below);
      if (!__any_sync(~0u, stop & ~found)) break;
    }
    return found;
  };

  uint32_t again = 0;
  int last = -1;
  bool token_again = false;
  for (uint32_t rest = bad; rest != 0; rest &= rest - 1) {
    const int bit = __ffs(rest) - 1, tok = (r.first + bit) / r.group;
    if (tok != last) {
      last = tok;
      const int64_t beg = begin_of(r.place0 + tok), end = end_of(r.place0 + tok);
      const bool empty = end <= beg;
      uint32_t masked = bad_columns(r.lo, empty || beg > r.hi ? r.hi : beg, false, ~0u);
      if (!empty) {
        masked |= bad_columns(end > r.lo ? end : r.lo, r.hi, false, ~0u);
        if (__any_sync(~0u, masked)) masked &= ~bad_columns(beg, end, true, masked);
      }
      token_again = __any_sync(~0u, masked);
    }
    if (token_again) again |= 1u << bit;
  }

  const float scale_log2 = a.scale * 1.4426950408889634f;
  while (again != 0) {
    // Lane 4 i keeps the score and the statistics of row i of the eight.
    int64_t beg = 0, end = 0, q_at = -1, out_at = -1;
    {
      uint32_t rest = again;
      for (int i = 0; i < lane / 4; ++i) rest &= rest - 1;
      if (rest != 0) {
        const int row = r.first + __ffs(rest) - 1, tok = row / r.group;
        const int head = r.head * r.group + row - tok * r.group;
        beg = begin_of(r.place0 + tok);
        end = end_of(r.place0 + tok);
        q_at = (r.row0 + tok) * a.q_token + head * a.q_head;
        out_at = (r.row0 + tok) * a.o_token + head * a.o_head;
      }
      for (int i = 0; i < kGroup; ++i) again &= again - 1;
    }
    float q[kGroup][C], acc[kGroup][C];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const int64_t at = __shfl_sync(~0u, q_at, 4 * i);
#pragma unroll
      for (int x = 0; x < C; ++x) {
        q[i][x] = at >= 0 && live ? to_f32(static_cast<const T*>(a.q)[at + e0 + x]) : 0.0f;
        acc[i][x] = 0.0f;
      }
    }
    float m = -INFINITY, l = 0.0f;
    int64_t j_beg = end > beg ? beg : r.keys, j_end = end > beg ? end : 0;
#pragma unroll
    for (int o = 4; o < 32; o *= 2) {
      const int64_t b = __shfl_xor_sync(~0u, j_beg, o), e = __shfl_xor_sync(~0u, j_end, o);
      j_beg = b < j_beg ? b : j_beg;
      j_end = e > j_end ? e : j_end;
    }
#pragma unroll 1
    for (int64_t j0 = j_beg; j0 < j_end; j0 += kBatch) {
      Columns ck[kBatch], cv[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        int64_t k, v;
        const bool real = j0 + b < j_end && key_at(j0 + b, &k, &v);
        ck[b] = load(kb, k, real && live);
        cv[b] = load(vb, v, real && live);
      }
      float s[kBatch], top = m;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        float p8[kGroup], p4[4], p2[2];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          p8[i] = 0.0f;
#pragma unroll
          for (int x = 0; x < C; ++x) p8[i] = fmaf(q[i][x], to_f32(ck[b].x[x]), p8[i]);
        }
        // Half of the rows go to the lane's partner at every step, until the
        // lane's own is left, of which four lanes hold a quarter each.
        const bool h16 = lane & 16, h8 = lane & 8, h4 = lane & 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p4[i] = (h16 ? p8[i + 4] : p8[i]) + __shfl_xor_sync(~0u, h16 ? p8[i] : p8[i + 4], 16);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          p2[i] = (h8 ? p4[i + 2] : p4[i]) + __shfl_xor_sync(~0u, h8 ? p4[i] : p4[i + 2], 8);
        float dot = (h4 ? p2[1] : p2[0]) + __shfl_xor_sync(~0u, h4 ? p2[0] : p2[1], 4);
        dot += __shfl_xor_sync(~0u, dot, 2);
        dot += __shfl_xor_sync(~0u, dot, 1);
        const bool seen = j0 + b >= beg && j0 + b < end;
        s[b] = seen ? dot * scale_log2 : -INFINITY;
        top = fmaxf(top, s[b]);
      }
      const float base = top == -INFINITY ? 0.0f : top;
      const float fix = exp2f(m - base);
      m = top;
      l *= fix;
      float w[kBatch];  // -1: a key that the row does not see
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const bool seen = j0 + b >= beg && j0 + b < end;
        w[b] = seen ? exp2f(s[b] - base) : -1.0f;
        if (seen) l += w[b];
      }
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const float f = __shfl_sync(~0u, fix, 4 * i);
#pragma unroll
        for (int x = 0; x < C; ++x) acc[i][x] *= f;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const float wi = __shfl_sync(~0u, w[b], 4 * i);
#pragma unroll
          for (int x = 0; x < C; ++x) {
            const float sum = fmaf(wi, to_f32(cv[b].x[x]), acc[i][x]);
            acc[i][x] = wi == -1.0f ? acc[i][x] : sum;
          }
        }
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const int64_t at = __shfl_sync(~0u, out_at, 4 * i);
      const float f = __shfl_sync(~0u, inv, 4 * i);
      if (at < 0 || !live) continue;
#pragma unroll
      for (int x = 0; x < C; ++x) {
        if (a.out_dtype == PSPML_DTYPE_S8)
          static_cast<int8_t*>(a.out)[at + e0 + x] =
              quantise_s8(acc[i][x] * f, a.out_inv_scale, a.out_zero);
        else
          static_cast<T*>(a.out)[at + e0 + x] = from_f32<T>(acc[i][x] * f);
      }
    }
  }
}

}  // namespace pspml
