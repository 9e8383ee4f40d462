// attn_step.cu - attention of a few new tokens per sequence over the paged
// cache (single-token decoding), F16 and BF16.
//
// All query rows that share a key head (new tokens x heads of its group, at
// most 16) form one 16-row tile, so every key and value is read from HBM
// once: 2 * keys * dim * 2 bytes a key head against 4 * 16 * dim flops a key
// even with padded rows, which keeps the kernel bound by the cache's bytes;
// m16n8k16 MMAs cover the padding's arithmetic many times over, and a
// 128-row tcgen05 tile would only add the 112 empty rows' softmax.
//
// Work is the list of (sequence, key head, 64 keys) tiles, counted on the
// device from the lengths and cut into equal contiguous shares, one per CTA:
// ragged batches stay balanced and one long sequence uses every SM.  A CTA
// walks its share with a ring of cp.async stages per warp (16 keys of the
// tile each, no barrier in the loop), a running maximum and sum in
// registers, and joins its warps where a (sequence, key head) ends.  Where a
// share cuts one, the pieces go to the workspace as unnormalised sums with
// their maximum and sum, and the CTA that arrives last joins them in order:
// the same bits on every call.  With several new tokens, rows that come out
// non-finite are looked at again (attn_rows.cuh).
//
// On a B200, cold, 32 query and 8 key heads of 128, BF16: one token over
// 131077 keys 89 us (537 MB, 6.0 TB/s); one token of each of 64 sequences of
// up to 8192 keys 207 us (1.19 GB, 5.7 TB/s).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "attention.h"
#include "attn_rows.cuh"
#include "ptx.cuh"

namespace pspml {

namespace {

constexpr int kStepThreads = 128;
constexpr int kStepWarps = 4;
constexpr int kStepTile = 64;   // keys, 16 per warp
constexpr int kStepRows = 16;
constexpr int kStepCtasPerSm = 2;
constexpr int kJoinDepth = 16;    // pieces whose loads are in flight in a join
// One token over 63776 keys of one key head takes 39 us at 2, 27 at 8, 28 at
// 32 and 33 with a piece on every CTA; over 25291 keys of two key heads 22, 16,
// 14 and 20 (with the launch, cold caches).
constexpr float kPieceTiles = 32;
// Segments of so few tiles are not cut: a cut costs about 3 us, a tile 0.3 (one
// token of 68 sequences of up to 353 keys: 16 us cut, 14 whole).
constexpr int kWholeTiles = 8;
static_assert(kStepCtasPerSm * kStepRows <= 256, "pieces fit the attention workspace");

struct StepArgs {
  AttnArgs a;
  float* part_o;       // [2 * ctas][16][DP]
  float2* part_ml;     // [2 * ctas][16]
  unsigned* arrived;   // [ctas], zero between calls
  float scale_log2;
  int32_t group;
};

template <int DP>
struct StepShape {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kChunks = DP / 8;               // 16-byte chunks a row
  static constexpr int kHalf = 16 * kRowBytes;         // one warp's K (or V) of a stage
  static constexpr int kStageBytes = 2 * kHalf;
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int kRing = kStages * kStageBytes;  // per warp
  static constexpr int kJoinBytes = 2 * kStepRows * DP * 4;
  static constexpr int kSmem = kStepWarps * kRing + kJoinBytes;
  static constexpr int kNB = DP / 8;                   // 8-wide output blocks
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  const int bytes = real ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Tiles of one sequence and key head, and where its keys begin and end.
struct StepSeq {
  int64_t begin, rows;        // rows: at most max_new
  int64_t keys;               // one past the last key that any of these rows sees
  int64_t place0;             // position of row 0
  int64_t lo;                 // first key any row sees
  int64_t first_tile;
  int64_t tiles;              // 0 only when there is no row
};
__device__ __forceinline__ StepSeq step_seq(const StepArgs& p, int s) {
  const SeqSpan sp = seq_span(p.a, s);
  StepSeq r;
  r.begin = sp.begin;
  r.place0 = sp.keys - sp.rows;
  r.rows = sp.rows < p.a.max_new ? sp.rows : p.a.max_new;
  // The keys of rows past max_new are not seen, so they are not multiplied
  // either: a single row (kMulti false) relies on it.
  const int64_t seen = r.place0 + r.rows;
  r.keys = !p.a.causal || seen > sp.keys ? sp.keys : (seen < 0 ? 0 : seen);
  r.lo = 0;
  if (p.a.window > 0 && r.place0 - p.a.window + 1 > 0) r.lo = r.place0 - p.a.window + 1;
  r.first_tile = r.lo / kStepTile;
  const int64_t n = (r.keys + kStepTile - 1) / kStepTile - r.first_tile;
  r.tiles = r.rows <= 0 ? 0 : (n < 1 ? 1 : n);
  return r;
}

// A position in the CTA's share.
struct StepCursor {
  StepSeq q;
  int s, head;
  int64_t tile;   // within the sequence and head
};
__device__ __forceinline__ void step_next_seq(const StepArgs& p, StepCursor& c) {
  do {
    if (++c.s >= p.a.sequences) return;
    c.q = step_seq(p, c.s);
  } while (c.q.tiles == 0);
}
__device__ __forceinline__ void step_advance(const StepArgs& p, StepCursor& c) {
  if (++c.tile < c.q.tiles) return;
  c.tile = 0;
  if (++c.head < p.a.kv_heads) return;
  c.head = 0;
  step_next_seq(p, c);
}

// First tile of CTA c's share; in 32 bits, a fraction of the time, when the
// product fits.
__device__ __forceinline__ int64_t share_of(unsigned c, int64_t total, int64_t ctas) {
  if (total < (1 << 21))  // at most 1024 CTAs
    return c * static_cast<uint32_t>(total) / static_cast<uint32_t>(ctas);
  return static_cast<int64_t>(c) * total / ctas;
}

// Writes a row pair's two neighbouring outputs.
template <typename T>
__device__ __forceinline__ void store2(const AttnArgs& a, int64_t at, float x, float y) {
  if (a.out_dtype == PSPML_DTYPE_S8) {
    char2 c;
    c.x = quantise_s8(x, a.out_inv_scale, a.out_zero);
    c.y = quantise_s8(y, a.out_inv_scale, a.out_zero);
    *reinterpret_cast<char2*>(static_cast<int8_t*>(a.out) + at) = c;
  } else {
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at) = pack2<T>(x, y);
  }
}

// kMulti: more than one new token a sequence, whose rows see different keys.
template <typename T, int DP, bool kMulti>
__global__ void __launch_bounds__(kStepThreads, kStepCtasPerSm) k_attn_step(const __grid_constant__ StepArgs p) {
  using Sh = StepShape<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_sum[kStepWarps];
  __shared__ int s_live[kStepWarps], s_longest[kStepWarps];
  __shared__ int64_t s_begin, s_end;
  __shared__ int s_seq;
  __shared__ int64_t s_base;
  __shared__ StepSeq s_first;
  __shared__ float s_m[kStepWarps][kStepRows], s_l[kStepWarps][kStepRows];
  __shared__ float2 s_join[kStepRows];
  __shared__ int s_last;
  __shared__ int s_bad;     // an output was not finite
  __shared__ int s_joined;  // bits: the cut segment at the share's begin, at its end
  const AttnArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  // Tiles before each thread's run of sequences, and in all.  One sequence a
  // thread at most is the usual case: its numbers are read once.
  const int per = (a.sequences + kStepThreads - 1) / kStepThreads;
  const int q0 = tid * per;
  const int q1 = min(a.sequences, q0 + per);
  int64_t mine = 0;
  int rows_seqs = 0;  // sequences with rows
  int64_t most = 0;   // tiles of the longest one
  StepSeq own{};
  for (int s = q0; s < q1; ++s) {
    own = step_seq(p, s);
    mine += own.tiles * a.kv_heads;
    rows_seqs += own.tiles > 0;
    most = own.tiles > most ? own.tiles : most;
  }
  rows_seqs = __reduce_add_sync(~0u, rows_seqs);
  const int longest = __reduce_max_sync(~0u, static_cast<int>(most));
  int64_t scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t v = __shfl_up_sync(~0u, scan, o);
    if (lane >= o) scan += v;
  }
  if (tid == 0) s_bad = s_joined = 0;
  if (lane == 31) {
    s_sum[warp] = scan;
    s_live[warp] = rows_seqs;
    s_longest[warp] = longest;
  }
  __syncthreads();
  int64_t total = 0, before = scan - mine, segments = 0;
  bool uncut = true;
#pragma unroll
  for (int w = 0; w < kStepWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
    segments += s_live[w];
    uncut &= s_longest[w] <= kWholeTiles;
  }
  segments *= a.kv_heads;
  // CTAs in use: every one of them has a tile.  A segment of T tiles in c
  // pieces takes T / c tiles' time and then a join that grows with c, so c
  // grows with the root of T; kPieceTiles is measured.
  int64_t ctas = total < gridDim.x ? total : gridDim.x;
  if (!uncut) {
    const float best = ceilf(sqrtf(kPieceTiles * static_cast<float>(total) *
                                   static_cast<float>(segments)));
    if (best < static_cast<float>(ctas)) ctas = static_cast<int64_t>(best);
  }
  if (blockIdx.x >= ctas) return;
  int64_t w0 = share_of(blockIdx.x, total, ctas), w1 = share_of(blockIdx.x + 1, total, ctas);
  if (uncut) {
    // Short segments stay whole: the shares' ends move to the nearest one's.
    if (tid == 0) s_end = total;  // the last share's
    __syncthreads();
    for (int e = 0; e < 2; ++e) {
      const int64_t w = e ? w1 : w0;
      if (w < before || w >= before + mine) continue;
      int64_t at = before;
      int s = q0;
      StepSeq q = own;
      while (per > 1) {
        q = step_seq(p, s++);
        if (w < at + q.tiles * a.kv_heads) break;
        at += q.tiles * a.kv_heads;
      }
      const int64_t in = (w - at) % q.tiles;
      (e ? s_end : s_begin) = 2 * in < q.tiles ? w - in : w - in + q.tiles;
    }
    __syncthreads();
    w0 = s_begin;
    w1 = s_end;
    if (w0 >= w1) return;
  }
  if (w0 >= before && w0 < before + mine) {
    int64_t at = before;
    int s = q0;
    while (per > 1) {
      own = step_seq(p, s);
      const int64_t n = own.tiles * a.kv_heads;
      if (w0 < at + n) break;
      at += n;
      ++s;
    }
    s_first = own;
    s_seq = s;
    s_base = at;
  }
  // Columns past the head's size stay zero for the whole kernel.
  const uint32_t ring = smem_u32(smem) + warp * Sh::kRing;
  const int live = a.dim / 8;
  if (live < Sh::kChunks) {
    for (int i = lane; i < Sh::kRing / 16; i += 32)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + i * 16), "r"(0)
                   : "memory");
    __syncwarp();
  }
  __syncthreads();

  StepCursor cur;
  cur.s = s_seq;
  cur.q = s_first;
  {
    const int64_t at = w0 - s_base;
    cur.head = static_cast<int>(at >> 32 == 0 ? static_cast<uint32_t>(at) /
                                                    static_cast<uint32_t>(cur.q.tiles)
                                              : at / cur.q.tiles);
    cur.tile = at - cur.head * cur.q.tiles;
  }
  int64_t seg_first = w0 - cur.tile;  // the current segment's first tile in the whole list
  StepCursor ld = cur;

  // This lane loads for key row lane % 16 of the warp's 16: its page is
  // looked up one tile ahead of the copies that need it.
  const T* kb = static_cast<const T*>(a.k);
  const T* vb = static_cast<const T*>(a.v);
  int64_t row_off = -1;
  auto look_up = [&]() {
    const int64_t j = (ld.q.first_tile + ld.tile) * kStepTile + warp * 16 + (lane & 15);
    row_off = -1;
    if (j >= ld.q.lo && j < ld.q.keys) {
      const uint32_t i = static_cast<uint32_t>(j) / static_cast<uint32_t>(a.page_size);
      const int32_t page = a.pages[ld.s * a.pages_stride + i];
      if (page >= 0 && page < a.n_pages)
        row_off = page * a.page_stride +
                  (static_cast<uint32_t>(j) - i * static_cast<uint32_t>(a.page_size)) * a.kv_token +
                  ld.head * a.kv_head;
    }
  };
  auto issue = [&](int stage) {
    const uint32_t dst = ring + stage * Sh::kStageBytes;
    constexpr int kRowsPer = 32 / Sh::kChunks;
    const int c = lane % Sh::kChunks;
#pragma unroll
    for (int i = 0; i < 16 / kRowsPer; ++i) {
      const int r = i * kRowsPer + lane / Sh::kChunks;
      const int64_t off = __shfl_sync(~0u, row_off, r);
      if (c < live) {
        const uint32_t d = dst + r * Sh::kRowBytes + ((c ^ (r & 7)) * 16);
        const int64_t e = off < 0 ? 0 : off + c * 8;
        cp_async16(d, kb + e, off >= 0);
        cp_async16(d + Sh::kHalf, vb + e, off >= 0);
      }
    }
  };

  const int64_t steps = w1 - w0;
  int64_t issued = 0;
  look_up();
#pragma unroll 1
  for (int i = 0; i < Sh::kStages - 1; ++i) {
    if (issued < steps) {
      issue(i);
      ++issued;
      step_advance(p, ld);
      if (issued < steps) look_up();
    }
    cp_commit();
  }

  uint32_t qf[DP / 16][4];
  float o[Sh::kNB][4];
  float m[2], l[2];
  int64_t place[2];
  const int r0 = lane / 4;

  int stage = 0, fill = Sh::kStages - 1;
  bool fresh = true;
#pragma unroll 1
  for (int64_t step = 0; step < steps; ++step) {
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = r0 + 8 * x;
        const int tok = r / p.group;
        const bool real = tok < cur.q.rows;
        place[x] = cur.q.place0 + tok;
        m[x] = -INFINITY;
        l[x] = 0.0f;
        const T* src = static_cast<const T*>(a.q) +
                       (real ? (cur.q.begin + tok) * a.q_token +
                                   (cur.head * p.group + (r - tok * p.group)) * a.q_head
                             : 0);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int e = kk * 16 + 8 * y + 2 * (lane % 4);
            qf[kk][x + 2 * y] =
                real && e < a.dim ? *reinterpret_cast<const uint32_t*>(src + e) : 0u;
          }
      }
#pragma unroll
      for (int i = 0; i < Sh::kNB; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
    }

    if (issued < steps) {
      issue(fill);
      ++issued;
      step_advance(p, ld);
      if (issued < steps) look_up();
    }
    cp_commit();
    fill = fill + 1 == Sh::kStages ? 0 : fill + 1;
    cp_wait<Sh::kStages - 1>();
    __syncwarp();

    const uint32_t ks = ring + stage * Sh::kStageBytes;
    float sc[2][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) sc[0][x] = sc[1][x] = 0.0f;
    {
      const int key = (lane / 16) * 8 + lane % 8, odd = (lane / 8) & 1;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t b[4];
        ldsm4(ks + key * Sh::kRowBytes + (((2 * kk + odd) ^ (key & 7)) * 16), b);
        mma16816<T>(sc[0], qf[kk], b[0], b[1]);
        mma16816<T>(sc[1], qf[kk], b[2], b[3]);
      }
    }
    const int64_t j0 = (cur.q.first_tile + cur.tile) * kStepTile + warp * 16;
    const int64_t last_place = cur.q.place0 + cur.q.rows - 1;
    const bool edge = j0 + 16 > cur.q.keys || (a.causal && j0 + 15 > cur.q.place0) ||
                      (a.window > 0 && j0 <= last_place - a.window);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        sc[n][x] *= p.scale_log2;
        if (edge) {
          const int64_t j = j0 + n * 8 + 2 * (lane % 4) + (x & 1);
          const int64_t pl = place[x / 2];
          if (j >= cur.q.keys || (a.causal && j > pl) || (a.window > 0 && j <= pl - a.window))
            sc[n][x] = -INFINITY;
        }
      }
    float pr[2][4];
    bool moved = false;
    float fix[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float t = fmaxf(fmaxf(sc[0][2 * x], sc[0][2 * x + 1]), fmaxf(sc[1][2 * x], sc[1][2 * x + 1]));
      t = fmaxf(t, __shfl_xor_sync(~0u, t, 1));
      t = fmaxf(t, __shfl_xor_sync(~0u, t, 2));
      const float m2 = fmaxf(m[x], t);
      const float base = m2 == -INFINITY ? 0.0f : m2;
      moved |= m2 != m[x];
      fix[x] = ex2(m[x] - base);
      m[x] = m2;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float e = ex2(sc[n][2 * x + y] - base);
          pr[n][2 * x + y] = e;
          sum += e;
        }
      l[x] = l[x] * fix[x] + sum;
    }
    if (__any_sync(~0u, moved)) {
#pragma unroll
      for (int i = 0; i < Sh::kNB; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] *= fix[x / 2];
    }
    uint32_t pf[4];
    pf[0] = pack2<T>(pr[0][0], pr[0][1]);
    pf[1] = pack2<T>(pr[0][2], pr[0][3]);
    pf[2] = pack2<T>(pr[1][0], pr[1][1]);
    pf[3] = pack2<T>(pr[1][2], pr[1][3]);
    {
      const int key = ((lane / 8) & 1) * 8 + lane % 8, right = lane / 16;
#pragma unroll
      for (int jj = 0; jj < DP / 16; ++jj) {
        uint32_t b[4];
        ldsm4_t(ks + Sh::kHalf + key * Sh::kRowBytes + (((2 * jj + right) ^ (key & 7)) * 16), b);
        mma16816<T>(o[2 * jj], pf, b[0], b[1]);
        mma16816<T>(o[2 * jj + 1], pf, b[2], b[3]);
      }
    }
    __syncwarp();  // the stage's rows are read before it is filled again
    stage = stage + 1 == Sh::kStages ? 0 : stage + 1;

    const bool seg_end = cur.tile + 1 == cur.q.tiles;
    if (seg_end || step + 1 == steps) {
      // Join the four warps: a common maximum per row, then the sums in a
      // fixed order (w2 and w3 into w0 and w1, w1 into w0).
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(~0u, l[x], 1);
        l[x] += __shfl_xor_sync(~0u, l[x], 2);
        if (lane % 4 == 0) s_m[warp][r0 + 8 * x] = m[x];
      }
      __syncthreads();
      float top[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = r0 + 8 * x;
        top[x] = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float f = ex2(m[x] - (top[x] == -INFINITY ? 0.0f : top[x]));
        l[x] *= f;
        if (lane % 4 == 0) s_l[warp][r] = l[x];
#pragma unroll
        for (int i = 0; i < Sh::kNB; ++i) {
          o[i][2 * x] *= f;
          o[i][2 * x + 1] *= f;
        }
      }
      float4* buf = reinterpret_cast<float4*>(smem + kStepWarps * Sh::kRing) +
                    (warp & 1) * (kStepRows * DP / 4);
      if (warp >= 2)
#pragma unroll
        for (int i = 0; i < Sh::kNB; ++i)
          buf[i * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
      __syncthreads();
      if (warp < 2)
#pragma unroll
        for (int i = 0; i < Sh::kNB; ++i) {
          const float4 v = buf[i * 32 + lane];
          o[i][0] += v.x;
          o[i][1] += v.y;
          o[i][2] += v.z;
          o[i][3] += v.w;
        }
      if (warp == 1)
#pragma unroll
        for (int i = 0; i < Sh::kNB; ++i)
          buf[i * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
      __syncthreads();
      const int64_t seg_tiles = cur.q.tiles;
      const bool whole = seg_first >= w0 && seg_end;
      const int rows = static_cast<int>(cur.q.rows) * p.group;
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (seg_first >= w0 ? 1 : 0);
      if (warp == 0) {
        const float4* other = reinterpret_cast<const float4*>(smem + kStepWarps * Sh::kRing) +
                              kStepRows * DP / 4;
        float inv[2], sum[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = r0 + 8 * x;
          sum[x] = (s_l[0][r] + s_l[2][r]) + (s_l[1][r] + s_l[3][r]);
          inv[x] = sum[x] == 0.0f ? 0.0f : 1.0f / sum[x];
        }
#pragma unroll
        for (int i = 0; i < Sh::kNB; ++i) {
          const float4 v = other[i * 32 + lane];
          o[i][0] += v.x;
          o[i][1] += v.y;
          o[i][2] += v.z;
          o[i][3] += v.w;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = r0 + 8 * x;
          if (r >= rows) continue;
          if (whole) {
            const int tok = r / p.group;
            const int64_t row = cur.q.begin + tok;
            const int h = cur.head * p.group + (r - tok * p.group);
            const int64_t at = row * a.o_token + h * a.o_head;
            float check = 0.0f;  // NaN once an output is not finite
#pragma unroll
            for (int i = 0; i < Sh::kNB; ++i) {
              const int e = i * 8 + 2 * (lane % 4);
              const float lo = o[i][2 * x] * inv[x], hi = o[i][2 * x + 1] * inv[x];
              if (e < a.dim) store2<T>(a, at + e, lo, hi);
              if (kMulti) check = fmaf(lo, 0.0f, fmaf(hi, 0.0f, check));
            }
            if (check != 0.0f) s_bad = 1;
            if (a.lse != nullptr && lane % 4 == 0)
              a.lse[row * a.q_heads + h] =
                  sum[x] == 0.0f ? -INFINITY : (log2f(sum[x]) + top[x]) * 0.69314718055994531f;
          } else {
            float* dst = p.part_o + (slot * kStepRows + r) * DP;
#pragma unroll
            for (int i = 0; i < Sh::kNB; ++i)
              *reinterpret_cast<float2*>(dst + i * 8 + 2 * (lane % 4)) =
                  make_float2(o[i][2 * x], o[i][2 * x + 1]);
            if (lane % 4 == 0) p.part_ml[slot * kStepRows + r] = make_float2(top[x], sum[x]);
          }
        }
      }
      if (!whole) {
        // The CTAs that hold pieces of this segment: tile f belongs to CTA
        // ((f + 1) * ctas - 1) / total.
        const int64_t c0 = ((seg_first + 1) * ctas - 1) / total;
        const int64_t c1 = ((seg_first + seg_tiles) * ctas - 1) / total;
        const int pieces = static_cast<int>(c1 - c0 + 1);
        if (warp == 0) {
          __threadfence();
          __syncwarp();
          if (lane == 0) {
            const unsigned n = atomicAdd(p.arrived + c0, 1u);
            s_last = n + 1 == static_cast<unsigned>(pieces);
            if (s_last) {
              p.arrived[c0] = 0;
              s_joined |= seg_first < w0 ? 1 : 2;
            }
          }
        }
        __syncthreads();
        if (s_last) {
          __threadfence();
          // Piece i is slot 2 c0 + 1 for i = 0, else 2 (c0 + i).
          auto slot_of = [&](int i) { return 2 * (c0 + i) + (i == 0 ? 1 : 0); };
          const int r = tid / 8;
          float mm = -INFINITY, ll = 0.0f;
          if (r < rows)
            for (int i = tid % 8; i < pieces; i += 8) {
              const float2 ml = __ldcg(p.part_ml + slot_of(i) * kStepRows + r);
              const float m2 = fmaxf(mm, ml.x);
              const float base = m2 == -INFINITY ? 0.0f : m2;
              ll = ll * ex2(mm - base) + ml.y * ex2(ml.x - base);
              mm = m2;
            }
#pragma unroll
          for (int x = 1; x < 8; x *= 2) {
            const float om = __shfl_xor_sync(~0u, mm, x), ol = __shfl_xor_sync(~0u, ll, x);
            const float m2 = fmaxf(mm, om);
            const float base = m2 == -INFINITY ? 0.0f : m2;
            ll = ll * ex2(mm - base) + ol * ex2(om - base);
            mm = m2;
          }
          if (tid % 8 == 0) s_join[r] = make_float2(mm == -INFINITY ? 0.0f : mm, ll);
          __syncthreads();
          for (int u = tid; u < rows * (DP / 4); u += kStepThreads) {
            const int rr = u / (DP / 4), e = (u % (DP / 4)) * 4;
            const float2 j = s_join[rr];
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll kJoinDepth
            for (int i = 0; i < pieces; ++i) {
              const int64_t at = slot_of(i) * kStepRows + rr;
              const float f = ex2(__ldcg(&p.part_ml[at].x) - j.x);
              const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * DP + e));
              acc.x = fmaf(v.x, f, acc.x);
              acc.y = fmaf(v.y, f, acc.y);
              acc.z = fmaf(v.z, f, acc.z);
              acc.w = fmaf(v.w, f, acc.w);
            }
            const float inv = j.y == 0.0f ? 0.0f : 1.0f / j.y;
            const int tok = rr / p.group;
            const int64_t row = cur.q.begin + tok;
            const int h = cur.head * p.group + (rr - tok * p.group);
            const int64_t at = row * a.o_token + h * a.o_head + e;
            acc.x *= inv;
            acc.y *= inv;
            acc.z *= inv;
            acc.w *= inv;
            if (e < a.dim) {
              store2<T>(a, at, acc.x, acc.y);
              store2<T>(a, at + 2, acc.z, acc.w);
            }
            if (kMulti &&
                fmaf(acc.x, 0.0f, fmaf(acc.y, 0.0f, fmaf(acc.z, 0.0f, acc.w * 0.0f))) != 0.0f)
              s_bad = 1;
            if (a.lse != nullptr && e == 0)
              a.lse[row * a.q_heads + h] =
                  j.y == 0.0f ? -INFINITY : (log2f(j.y) + j.x) * 0.69314718055994531f;
          }
        }
      }
      __syncthreads();  // the join buffers are free for the next segment
      seg_first += seg_tiles;
      fresh = true;
    }
    step_advance(p, cur);
  }
  cp_wait<0>();
  if constexpr (kMulti) {
    if (s_bad == 0) return;
    // Once more over the segments whose outputs this CTA wrote: here, so that
    // the loop above keeps its registers (391 us against 235 for 64 sequences
    // of up to 8192 keys with the call inside, and 225 without it: a single
    // token's rows see the same keys and do without).
    cur.s = s_seq;
    cur.q = s_first;
    cur.head = static_cast<int>((w0 - s_base) / cur.q.tiles);
    for (int64_t at = s_base + cur.head * cur.q.tiles; at < w1;) {
      const int64_t end = at + cur.q.tiles;
      if ((at >= w0 && end <= w1) || (s_joined & (at < w0 ? 1 : 2)) != 0) {
        AttnRows r;
        r.table = a.pages + cur.s * a.pages_stride;
        r.begin = 0;
        r.keys = r.hi = cur.q.keys;
        r.lo = cur.q.lo;
        r.row0 = cur.q.begin;
        r.place0 = cur.q.place0;
        r.head = cur.head;
        r.group = p.group;
        r.first = 0;
        const int rows = static_cast<int>(cur.q.rows) * p.group;
        attn_rows_again<T, DP>(a, r, ((1u << rows) - 1u) & (0xFu << (4 * warp)));
      }
      at = end;
      if (++cur.head == a.kv_heads) {
        cur.head = 0;
        step_next_seq(p, cur);
      }
    }
  }
}

template <typename T, int DP, bool kMulti>
cudaError_t step_launch(const StepArgs& p, int grid, cudaStream_t s) {
  using Sh = StepShape<DP>;
  static std::atomic<uint64_t> attr_done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if ((attr_done.load() & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(
        k_attn_step<T, DP, kMulti>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
    if (e != cudaSuccess) return e;
    attr_done.fetch_or(bit);
  }
  k_attn_step<T, DP, kMulti><<<grid, kStepThreads, Sh::kSmem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_step(const AttnArgs& a, const AttnWork& w, cudaStream_t s) {
  const int dp = a.dim <= 64 ? 64 : 128;
  const int grid = std::min(w.num_sms * kStepCtasPerSm, kAttnCounters);
  StepArgs p{};
  p.a = a;
  p.part_o = reinterpret_cast<float*>(w.base);
  p.part_ml = reinterpret_cast<float2*>(w.base + 2ull * grid * kStepRows * dp * sizeof(float));
  p.arrived = w.counters;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.group = a.q_heads / a.kv_heads;
  auto by_tokens = [&](auto type, auto size) {
    using T = decltype(type);
    constexpr int kDp = decltype(size)::value;
    return a.max_new > 1 ? step_launch<T, kDp, true>(p, grid, s)
                         : step_launch<T, kDp, false>(p, grid, s);
  };
  auto by_size = [&](auto type) {
    return dp == 64 ? by_tokens(type, std::integral_constant<int, 64>{})
                    : by_tokens(type, std::integral_constant<int, 128>{});
  };
  return a.dtype == PSPML_DTYPE_F16 ? by_size(__half{})
                                      : by_size(__nv_bfloat16{});
}

}  // namespace pspml
