// attn_tc.cu - attention over whole prompts and of chunks of new tokens over
// the paged cache on the tensor cores (tcgen05), F16 and BF16.
//
//   S = Q K^T,  P = exp2(c S - m),  O = P V / sum P,   c = scale * log2 e
//
// Rows of a tile are (token, head of the key head's group) pairs, 128 / group
// tokens a tile: the heads that share keys share their loads, short chunks
// fill a tile with heads, and the causal edge is a few tokens wide instead
// of 128.  A CTA takes two such tiles (A, B) against one stream of 128-key
// tiles, so that the tensor cores work on one tile while the softmax of the
// other runs:
//   warps 0-3, 4-7  softmax of A and B, one row per thread: S from tensor
//                   memory, running maximum and sum in registers, P back to
//                   tensor memory over S (as the A operand of P V); the
//                   output is rescaled only when the maximum has grown by
//                   more than 2^8 since the last time, by the same threads
//   warp 8          TMA loads: Q once, K and V tiles through a ring of slots
//   warp 9          one thread issues the MMAs: P V of a tile, then the next
//                   Q K^T of the same tile once P has been read (warps 10
//                   and 11 only fill the warpgroup)
// Tensor memory: S/P of A and B (128 columns each), O of A and B.
//
// Keys that no row of the CTA sees are not loaded; the values between such a
// key and the 16-key step of the P V product that holds it are zeroed in
// shared memory, since 0 * NaN would spread whatever they hold.  Rows that
// come out non-finite are looked at again (attn_rows.cuh), for what a key
// that some rows see did to those that do not.  Heads of fewer than DP
// elements are padded with zeros by TMA.
//
// A CTA stays for many items (a pair of tiles and a key head): the next one's
// loads and first scores run while this one ends.  Many items are handed out
// by a counter, within a sequence those with the most keys first.  Few items
// are cut: the list of all their key tiles is divided into equal shares, and
// where a share cuts an item the pieces go to the workspace, unnormalised, and
// the CTA that arrives last joins them in order, so the same call gives the
// same bits.
//
// What bounds it: the chain of one tile (scores 592 clocks and 270 until they
// are seen, softmax 2000 to 2250, the last half of P V and its completion 470)
// sets 3430 clocks a pair of key tiles against 2208 of tensor work; shared
// memory feeds the scores at its full 128 bytes a clock.  On a B200, BF16, 32
// query and 8 key heads of 128: 16384 tokens 1.73 ms alone (1.27 PFLOP/s) and
// 2.00 ms in a long row of passes, where power limits the clock; 17 packed
// prompts of up to 2048 tokens 148 us (0.70 PFLOP/s), 135 us with inputs that
// stay in L2.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "attention.h"
#include "attn_giveup.cuh"
#include "attn_rows.cuh"
#include "ptx.cuh"

namespace pspml {

namespace {

// Three warpgroups: 168 registers a thread at launch, of which the softmax
// groups take 200 and the third keeps 104 (128 * (2 * 200 + 104) = 384 * 168).
constexpr int kTcThreads = 384;
constexpr int kSoftmaxRegs = 200;
constexpr int kOtherRegs = 104;
constexpr int kKeys = 128;        // keys a tile
constexpr int kPieces = 2;        // in which P is handed to the MMA warp
// Calls of fewer items an SM count their key tiles, and are cut into equal
// shares if the longest item has kCutTiles more than a share.  Cutting costs a
// piece written and read per cut, about the time of as many tiles: 400 items
// of 7 tiles on average take 72 us whole and 104 us cut, 80 items of up to 94
// tiles 189 us whole and 131 us cut.
constexpr int kItemsPerSm = 2;
constexpr int kCutTiles = 6;
constexpr float kGrowLog2 = 8.0f; // largest stale maximum, as a power of two

struct TcArgs {
  AttnArgs a;
  float4* part_o;      // [2 * ctas][DP / 4][256]: a warp's rows side by side
  float2* part_ml;     // [2 * ctas][256]
  unsigned* arrived;   // [ctas]
  unsigned* next;      // first item that no CTA has taken, less the grid's size
  unsigned* done;      // CTAs that have finished
  unsigned* err;
  float scale_log2;
  int64_t items;       // pairs * key heads, at most
  int32_t group, tile_tokens, box_keys;
  int32_t wide_out;    // output rows start on 32-byte boundaries
  int32_t shares;      // equal shares of key tiles instead of whole items
};

template <int DP>
struct TcShape {
  static constexpr int kHalves = DP / 64;           // 128-byte swizzled halves of a row
  static constexpr int kTileBytes = 128 * DP * 2;   // Q tile, K or V slot
  static constexpr int kSlots = DP == 128 ? 5 : 8;
  static constexpr int kSmem = 1024 + (2 + kSlots) * kTileBytes;
  static constexpr uint32_t kCols = 512;
  static constexpr uint32_t kS = 0;                 // S/P of A, then of B
  static constexpr uint32_t kO = 256;               // O of A, then of B
};

// Two floats in one 64-bit register, and the packed arithmetic on them.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_get(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The CTA's state: kGaveUp once a wait has run out, and kRowsAgain for every
// warp that is doing rows again.
constexpr int kGaveUp = 1;
constexpr int kRowsAgain = 2;
__device__ __forceinline__ void tc_fail(unsigned* err, int* state, unsigned code) {
  atomicOr(state, kGaveUp);
  atomicCAS(err, 0u, code);
}
// The waits of ptx.cuh (kPoll: without the suspend-time hint), which end when
// the CTA has given up.  Rows done again hold the CTA's other warps up for as
// long as their keys take, seconds for a long context: no signal is lost, and
// the limit does not run meanwhile.
template <bool kPoll = false>
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, const int* state,
                                        uint64_t limit_ns = kWaitLimitNs) {
  auto passed = [&]() {
    return kPoll ? mbar_try_wait_poll(bar, parity) : mbar_try_wait(bar, parity);
  };
  if (passed()) return true;
  uint64_t t0 = global_timer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < (kPoll ? 64 : 32); ++i)
      if (passed()) return true;
    const int now = *static_cast<const volatile int*>(state);
    if (now != 0) {
      if (now & kGaveUp) return false;
      t0 = global_timer_ns();
    }
    if (global_timer_ns() - t0 > limit_ns) return false;
  }
}

// Piece h of tile t's P is handed from its four softmax warps to the MMA warp
// at a hardware barrier: polls of an mbarrier would take issue slots from the
// two softmax warps on the MMA warp's scheduler, which set the pace (2121 us
// against 1854 at 16384 tokens and 32 heads with tight and with rare polls).
// These waits have no limit; attn_giveup.cuh says why they end.  `n`: key tiles
// of tile t before this one.
__device__ __forceinline__ void prob_arrive(int t, int h, uint32_t n) {
  asm volatile("bar.arrive %0, 160;" ::"r"(prob_barrier(t, h, n)) : "memory");
}
__device__ __forceinline__ void prob_meet(int t, int h, uint32_t n) {
  asm volatile("bar.sync %0, 160;" ::"r"(prob_barrier(t, h, n)) : "memory");
}

// Eight neighbouring outputs of a row.
template <typename T>
__device__ __forceinline__ void store8(const AttnArgs& a, int64_t at, const float* v) {
  if (a.out_dtype == PSPML_DTYPE_S8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[i] |= static_cast<uint32_t>(static_cast<uint8_t>(
                    quantise_s8(v[4 * i + k], a.out_inv_scale, a.out_zero)))
                << (8 * k);
    }
    *reinterpret_cast<uint2*>(static_cast<int8_t*>(a.out) + at) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                   pack2<T>(v[6], v[7]));
  }
}

// The n lowest bits, n cut to 0 .. 32.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u);
}

// Sixteen (or, at the end of a head, eight) neighbouring outputs of a row; as
// one 32-byte sector where the view's alignment allows it.
template <typename T>
__device__ __forceinline__ void store16(const AttnArgs& a, int64_t at, const float* v, bool both,
                                        bool wide) {
  if (both && wide && a.out_dtype != PSPML_DTYPE_S8) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    st_global_v8(static_cast<T*>(a.out) + at, make_uint4(w[0], w[1], w[2], w[3]),
                 make_uint4(w[4], w[5], w[6], w[7]));
  } else {
    store8<T>(a, at, v);
    if (both) store8<T>(a, at + 8, v + 8);
  }
}

// Rows, positions and keys of a CTA's two tiles.
struct TcGeometry {
  int64_t row0;     // first row of the pair in q and out
  int64_t keys;     // of the sequence
  int64_t place0;   // position of the pair's first token
  int64_t lo;       // first key that any row sees
  int64_t start;    // first key of key tile 0
  int64_t hi_all;   // one past the last key that any row sees
  int tokens0, tokens1;  // of tile A and B
  int tiles0, tiles1;    // key tiles of A and B
};
__device__ __forceinline__ unsigned tc_pairs(const TcArgs& p, const SeqSpan& sp) {
  const int64_t rows = p.a.paged && sp.rows > p.a.max_new ? p.a.max_new : sp.rows;
  const unsigned pair_tokens = 2u * p.tile_tokens;
  return (static_cast<unsigned>(rows) + pair_tokens - 1) / pair_tokens;
}
// Pair `idx` of the call, found by one warp: the sequences' pairs are counted
// 32 sequences at a time.  Within a sequence the last tokens come first, so
// that the pairs with the most keys start first.  False past the last pair.
__device__ __forceinline__ bool tc_locate(const TcArgs& p, int64_t idx, int lane, int* seq,
                                          int64_t* pair, SeqSpan* span) {
  for (int s0 = 0; s0 < p.a.sequences; s0 += 32) {
    const int s = s0 + lane;
    SeqSpan sp{0, 0, 0};
    unsigned mine = 0;
    if (s < p.a.sequences) {
      sp = seq_span(p.a, s);
      mine = tc_pairs(p, sp);
    }
    unsigned scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned v = __shfl_up_sync(~0u, scan, o);
      if (lane >= o) scan += v;
    }
    const unsigned all = __shfl_sync(~0u, scan, 31);
    if (idx < all) {
      const int at = __ffs(__ballot_sync(~0u, idx < scan)) - 1;
      *seq = s0 + at;
      *pair = static_cast<int64_t>(__shfl_sync(~0u, scan, at)) - 1 - idx;
      span->begin = __shfl_sync(~0u, sp.begin, at);
      span->keys = __shfl_sync(~0u, sp.keys, at);
      span->rows = __shfl_sync(~0u, sp.rows, at);
      return true;
    }
    idx -= all;
  }
  return false;
}
__device__ __forceinline__ TcGeometry tc_geometry(const TcArgs& p, const SeqSpan& sp,
                                                  int64_t pair) {
  const AttnArgs& a = p.a;
  const int64_t rows = a.paged && sp.rows > a.max_new ? a.max_new : sp.rows;
  const int64_t tok0 = pair * 2 * p.tile_tokens, left = rows - tok0;  // left: at least 1
  TcGeometry g;
  g.row0 = sp.begin + tok0;
  g.keys = sp.keys;
  g.place0 = sp.keys - sp.rows + tok0;
  g.tokens0 = static_cast<int>(left < p.tile_tokens ? left : p.tile_tokens);
  g.tokens1 = static_cast<int>(left < 2 * p.tile_tokens ? left : 2 * p.tile_tokens) - g.tokens0;
  g.lo = a.window > 0 && g.place0 - a.window + 1 > 0 ? g.place0 - a.window + 1 : 0;
  g.start = g.lo / kKeys * kKeys;
  int64_t hi0 = sp.keys, hi1 = sp.keys;
  if (a.causal) {
    const int64_t e0 = g.place0 + g.tokens0, e1 = g.place0 + p.tile_tokens + g.tokens1;
    if (e0 < hi0) hi0 = e0;
    if (e1 < hi1) hi1 = e1;
  }
  g.hi_all = g.tokens1 > 0 ? hi1 : hi0;
  g.tiles0 = hi0 > g.lo ? static_cast<int>((hi0 - g.start + kKeys - 1) / kKeys) : 0;
  g.tiles1 =
      g.tokens1 > 0 && hi1 > g.lo ? static_cast<int>((hi1 - g.start + kKeys - 1) / kKeys) : 0;
  return g;
}

// Key tiles that an item counts for: one at least, since its rows have to be
// written even when they see no key.
__device__ __forceinline__ int tc_units(const TcGeometry& g) {
  return max(1, max(g.tiles0, g.tiles1));
}
// The sum of `v` over the threads before this one in the block; `all`: over
// the block.
__device__ __forceinline__ int tc_scan(int v, int tid, int* warp_sums, int* all) {
  const int lane = tid % 32;
  int scan = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int x = __shfl_up_sync(~0u, scan, o);
    if (lane >= o) scan += x;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 31) warp_sums[tid / 32] = scan;
  __syncthreads();
  int before = 0;
  *all = 0;
#pragma unroll
  for (int w = 0; w < kTcThreads / 32; ++w) {
    if (w < tid / 32) before += warp_sums[w];
    *all += warp_sums[w];
  }
  return before + scan - v;
}
// The last of the n ascending numbers that is at most x, which the first is.
__device__ __forceinline__ int tc_find(const int* a, int n, int64_t x, int per) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (static_cast<int64_t>(a[mid]) * per <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// What a CTA's warps need to know of one item, or of its part of one.
struct TcItem {
  int64_t row0, place0, keys, lo, start, hi_all;
  int32_t tokens[2];   // of tile A and B
  int32_t n[2];        // key tiles of A and B in this part
  int32_t j0;          // the part's first key tile
  int32_t seq, head;
  int32_t pieces;      // CTAs that share the item
  int32_t first_cta;   // of them
  int32_t end;         // no more items
};
constexpr int kMinShare = 4;     // key tiles of a share, at least
// Where a CTA's share of the key tiles begins and ends.
struct TcShare {
  int64_t total = 0, at = 0, stop = 0;  // key tiles of all items; this CTA's
  int ctas = 0;                         // CTAs in use; 0: items are handed out whole
  int seq = 0, head = 0, tile = 0;
  int64_t pair = 0;
  SeqSpan span{0, 0, 0};
};
// Of the wait for the next item, and of the loader's for a record: longer than
// any wait within an item, of which the others wait for several.
constexpr uint64_t kItemLimitNs = 5 * kWaitLimitNs;
static_assert(kPieces == 2, "prob_barrier's layout");

template <typename T, int DP>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_attn_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcArgs p) {
  using Sh = TcShape<DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, q_empty, landed, s_full[2], o_done[2], drain;
  __shared__ uint64_t kv_full[Sh::kSlots], kv_empty[Sh::kSlots];
  __shared__ uint64_t item_full[2], item_empty[2];
  __shared__ TcItem items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int state_word;
  __shared__ int book;  // of items (attn_giveup.cuh)
  __shared__ int s_last, s_longest, s_scan[kTcThreads / 32];
  const AttnArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  int* const state = &state_word;
  auto gave_up = [&]() { return (*static_cast<volatile int*>(state) & kGaveUp) != 0; };
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* sq = smem;
  uint8_t* slots = smem + 2 * Sh::kTileBytes;

  if (tid == 0) {
    state_word = 0;
    book = 0;
    s_longest = 0;
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    mbar_init(&landed, 1);
    mbar_init(&drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 9);  // the MMA warp and eight softmax warps
    }
    for (int i = 0; i < Sh::kSlots; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 8) {
    if (lane == 0) {
      tma_prefetch_desc(&map_q);
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
    tmem_alloc(&tmem_slot, Sh::kCols);
    tmem_relinquish();
  }
  // Few items, so fewer sequences and pairs than kItemsPerSm an SM (some 11000
  // pairs if `starts` decreases against its contract, 44 KB): their key tiles
  // are counted, with room for the tiles as scratch.  Cutting pays where one item outlasts an equal share by more
  // than the pieces cost.
  TcShare share;
  bool more = p.items > gridDim.x;  // than one item a CTA, handed out by the counter
  if (p.shares) {
    int* const first_pair = reinterpret_cast<int*>(sq);  // of each sequence
    int pairs = 0, all;
    for (int s0 = 0; s0 < a.sequences; s0 += kTcThreads) {
      const int s = s0 + tid;
      const int mine =
          s < a.sequences ? static_cast<int>(tc_pairs(p, seq_span(a, s))) : 0;
      const int before = tc_scan(mine, tid, s_scan, &all);
      if (s < a.sequences) first_pair[s] = pairs + before;
      pairs += all;
    }
    if (tid == 0) first_pair[a.sequences] = pairs;
    __syncthreads();
    int* const first_tile = first_pair + a.sequences + 1;  // of each pair, for one key head
    int tiles = 0, longest = 0;
    for (int i0 = 0; i0 < pairs; i0 += kTcThreads) {
      const int i = i0 + tid;
      int units = 0;
      if (i < pairs) {
        const int s = tc_find(first_pair, a.sequences, i, 1);
        units = tc_units(tc_geometry(p, seq_span(a, s), first_pair[s + 1] - 1 - i));
      }
      const int before = tc_scan(units, tid, s_scan, &all);
      if (i < pairs) first_tile[i] = tiles + before;
      tiles += all;
      longest = max(longest, units);
    }
    if (tid == 0) first_tile[pairs] = tiles;
    longest = __reduce_max_sync(~0u, longest);
    if (lane == 0) atomicMax(&s_longest, longest);
    __syncthreads();
    const int64_t total = static_cast<int64_t>(tiles) * a.kv_heads;
    if (s_longest > total / gridDim.x + kCutTiles) {
      more = false;
      share.total = total;
      const int64_t wanted = (total + kMinShare - 1) / kMinShare;
      share.ctas = static_cast<int>(wanted < gridDim.x ? wanted : gridDim.x);
      if (blockIdx.x < share.ctas) {
        share.at = blockIdx.x * total / share.ctas;
        share.stop = (blockIdx.x + 1) * total / share.ctas;
        const int i = tc_find(first_tile, pairs, share.at, a.kv_heads);
        const int units = first_tile[i + 1] - first_tile[i];
        const int64_t in = share.at - static_cast<int64_t>(first_tile[i]) * a.kv_heads;
        share.head = static_cast<int>(in / units);
        share.tile = static_cast<int>(in - static_cast<int64_t>(share.head) * units);
        share.seq = tc_find(first_pair, a.sequences, i, 1);
        share.pair = first_pair[share.seq + 1] - 1 - i;
        share.span = seq_span(a, share.seq);
      }
    }
    fence_async_smem();  // the scratch is read before TMA writes over it
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // Item `it` of this CTA, published by warp 8.  Every warp takes the same
  // items, and whoever has taken one walks all of it.
  auto take = [&](int it) -> const TcItem* {
    if (!__all_sync(~0u, tc_wait(&item_full[it & 1], static_cast<uint32_t>((it >> 1) & 1), state,
                                 kItemLimitNs))) {
      bool closed = false;
      if (lane == 0) {
        closed = item_close(&book, it);
        if (closed) tc_fail(p.err, state, kDevErrEpiWait);
      }
      closed = __any_sync(~0u, closed);
      __syncwarp();  // the record, if it is there, is there for every lane
      if (closed) return nullptr;
    }
    return &items[it & 1];
  };
  // Keys of tile j that some row sees: [v_lo, v_hi) of its 128.
  auto v_lo = [](int64_t lo, int64_t start, int j) {
    const int64_t x = lo - (start + static_cast<int64_t>(j) * kKeys);
    return x > 0 ? static_cast<int>(x) : 0;
  };
  auto v_hi = [](int64_t hi_all, int64_t start, int j) {
    const int64_t x = hi_all - (start + static_cast<int64_t>(j) * kKeys);
    return x < kKeys ? static_cast<int>(x) : kKeys;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // ------------------------------------------------- items and TMA loads
      const int boxes = kKeys / p.box_keys;  // one per lane
      int slot = 0, landings = 0, issued = 0, q_loads = 0;
      uint32_t phase = 0;
      bool ok = true;
      int64_t next = blockIdx.x;  // handed out: the item
      const bool cut = share.ctas > 0;
      int seq = share.seq, head = share.head, tile = share.tile;
      int64_t pair = share.pair, at = share.at;
      SeqSpan span = share.span;
      for (int it = 0;; ++it) {
        TcItem* const d = &items[it & 1];
        if (it >= 2 && !tc_wait(&item_empty[it & 1], static_cast<uint32_t>(((it >> 1) - 1) & 1),
                                state, kItemLimitNs)) {
          tc_fail(p.err, state, kDevErrTmaWait);
          ok = false;
        }
        if (!__all_sync(~0u, ok && !gave_up())) {
          // The record may still be that of an item that some warp has not taken.
          if (lane == 0) item_close(&book, it);
          break;
        }
        bool have = at < share.stop;
        if (!cut) {
          head = static_cast<int>(next % a.kv_heads);
          have = next < p.items && tc_locate(p, next / a.kv_heads, lane, &seq, &pair, &span);
        }
        if (!have) {
          if (lane == 0) {
            d->end = 1;
            if (item_publish(&book, it)) mbar_arrive(&item_full[it & 1]);
          }
          break;
        }
        const TcGeometry g = tc_geometry(p, span, pair);
        const int64_t lo = g.lo, start = g.start, hi_all = g.hi_all;
        const int units = tc_units(g), j0 = tile;
        int j1 = units, pieces = 1, first_cta = 0;
        if (cut) {
          if (share.stop - at < j1 - j0) j1 = j0 + static_cast<int>(share.stop - at);
          if (j0 > 0 || j1 < units) {
            // Tile f of the list belongs to CTA ((f + 1) * ctas - 1) / total.
            const int64_t f = at - j0;
            first_cta = static_cast<int>(((f + 1) * share.ctas - 1) / share.total);
            pieces = static_cast<int>(((f + units) * share.ctas - 1) / share.total) - first_cta + 1;
          }
        }
        const int n0 = max(0, min(j1, g.tiles0) - j0), n1 = max(0, min(j1, g.tiles1) - j0);
        const int n = max(n0, n1);
        if (lane == 0) {
          d->row0 = g.row0;
          d->place0 = g.place0;
          d->keys = g.keys;
          d->lo = lo;
          d->start = start;
          d->hi_all = hi_all;
          d->tokens[0] = g.tokens0;
          d->tokens[1] = g.tokens1;
          d->n[0] = n0;
          d->n[1] = n1;
          d->j0 = j0;
          d->seq = seq;
          d->head = head;
          d->pieces = pieces;
          d->first_cta = first_cta;
          d->end = 0;
          ok = item_publish(&book, it);
          if (ok) mbar_arrive(&item_full[it & 1]);
        }
        if (!__all_sync(~0u, ok)) break;
        // The next item: asked for now, looked at when this one's loads are out.
        unsigned taken = 0;
        if (more && lane == 0) taken = atomicAdd(p.next, 1u);

        const int32_t* table = a.paged ? a.pages + seq * a.pages_stride : nullptr;
        auto page_of = [&](int j) -> int {
          const int64_t key = start + static_cast<int64_t>(j) * kKeys + lane * p.box_keys;
          if (!a.paged || lane >= boxes || key + p.box_keys <= lo || key >= hi_all) return -1;
          return table[static_cast<uint32_t>(key) / static_cast<uint32_t>(a.page_size)];
        };
        int page = n > 0 ? page_of(j0) : -1;
        if (n > 0) {
          const uint32_t q_phase = static_cast<uint32_t>((q_loads - 1) & 1);
          if (q_loads > 0 && !tc_wait(&q_empty, q_phase, state)) {
            tc_fail(p.err, state, kDevErrTmaWait);
            ok = false;
          }
          __syncwarp();
          if (lane == 0) {
            const int boxes_q = ((n0 > 0) + (n1 > 0)) * Sh::kHalves;
            mbar_arrive_expect_tx(
                &q_full, static_cast<uint32_t>(boxes_q * p.tile_tokens * p.group * 128));
            for (int t = 0; t < 2; ++t) {
              if ((t == 0 ? n0 : n1) == 0) continue;
              for (int h = 0; h < Sh::kHalves; ++h)
                tma_load_4d(sq + t * Sh::kTileBytes + h * 16384, &map_q, &q_full, h * 128, 0, head,
                            static_cast<int32_t>(g.row0 + t * p.tile_tokens));
            }
          }
          ++q_loads;
        }
        for (int j = j0; j < j0 + n && ok; ++j) {
          const int64_t kb = start + static_cast<int64_t>(j) * kKeys;
          const int lo_k = v_lo(lo, start, j), hi_k = v_hi(hi_all, start, j);
          const int first = lane * p.box_keys;
          const bool load = lane < boxes && first < hi_k && first + p.box_keys > lo_k;
          const int n_load = __popc(__ballot_sync(~0u, load));
          const uint32_t bytes = static_cast<uint32_t>(n_load * p.box_keys * 128 * Sh::kHalves);
          const int next_page = j + 1 < j0 + n ? page_of(j + 1) : -1;
          const int32_t c2 = a.paged ? static_cast<int32_t>(static_cast<uint32_t>(kb + first) %
                                                            static_cast<uint32_t>(a.page_size))
                                     : static_cast<int32_t>(span.begin + kb + first);
          const int32_t c3 = a.paged ? page : 0;
          for (int which = 0; which < 2; ++which) {
            const bool got = tc_wait(&kv_empty[slot], phase ^ 1u, state);
            if (!got) tc_fail(p.err, state, kDevErrTmaWait);
            if (!__all_sync(~0u, got)) {
              ok = false;
              break;
            }
            uint8_t* dst = slots + slot * Sh::kTileBytes;
            const bool mend = which == 1 && ((lo_k | hi_k) & 15) != 0;
            uint64_t* bar = mend ? &landed : &kv_full[slot];
            if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (load)
              for (int h = 0; h < Sh::kHalves; ++h)
                tma_load_4d(dst + h * 16384 + first * 128, which ? &map_v : &map_k, bar, h * 128,
                            head, c2, c3);
            __syncwarp();
            if (mend) {
              if (!tc_wait(&landed, static_cast<uint32_t>(landings & 1), state)) {
                tc_fail(p.err, state, kDevErrTmaWait);
                ok = false;
              }
              ++landings;
              const int a0 = lo_k & ~15, a1 = (hi_k + 15) & ~15;
              const int dead = (lo_k - a0) + (a1 - hi_k);
              for (int u = lane; u < dead * 8 * Sh::kHalves; u += 32) {
                const int i = u / (8 * Sh::kHalves), c = u % (8 * Sh::kHalves);
                const int r = i < lo_k - a0 ? a0 + i : hi_k + (i - (lo_k - a0));
                *reinterpret_cast<uint4*>(dst + (c / 8) * 16384 + r * 128 + (c % 8) * 16) =
                    make_uint4(0, 0, 0, 0);
              }
              fence_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&kv_full[slot]);
            }
            ++issued;
            if (++slot == Sh::kSlots) {
              slot = 0;
              phase ^= 1u;
            }
          }
          ok = __all_sync(~0u, ok);
          page = next_page;
        }
        if (!cut) {
          next = more ? static_cast<int64_t>(__shfl_sync(~0u, taken, 0)) + gridDim.x : p.items;
          continue;
        }
        at += j1 - j0;
        tile = j1 < units ? j1 : 0;
        if (tile == 0 && ++head == a.kv_heads) {
          head = 0;
          if (--pair < 0)
            while (++seq < a.sequences) {
              span = seq_span(a, seq);
              pair = static_cast<int64_t>(tc_pairs(p, span)) - 1;
              if (pair >= 0) break;
            }
        }
      }
      if (__any_sync(~0u, !ok || gave_up())) {  // the copies in flight land before the CTA leaves
        if (q_loads > 0) mbar_wait(&q_full, static_cast<uint32_t>((q_loads - 1) & 1), nullptr);
        if (landings > 0) mbar_wait(&landed, static_cast<uint32_t>((landings - 1) & 1), nullptr);
        for (int i = issued > Sh::kSlots ? issued - Sh::kSlots : 0; i < issued; ++i)
          mbar_wait(&kv_full[i % Sh::kSlots], static_cast<uint32_t>((i / Sh::kSlots) & 1), nullptr);
      }
      __syncwarp();
    } else if (warp == 9) {
      // --------------------------------------------------------------- MMAs
      // The whole warp walks the loop and its waits; elect.sync names the one
      // lane that issues, which is how the compiler knows that the operands of
      // an MMA are one thread's and moves them to the tensor core directly.
      {
        constexpr int kFmt = std::is_same<T, __half>::value ? 0 : 1;
        const int k_steps = (a.dim + 15) / 16;
        const uint32_t id_qk = make_idesc_f16(128, kKeys, kFmt, 0);
        const uint32_t id_pv = make_idesc_f16(128, k_steps * 16, kFmt, 1);
        const uint32_t q_addr = smem_u32(sq), kv_addr = smem_u32(slots);
        // A wait that gives up only changes the state, after which every
        // other wait ends at once.
        auto wait = [&](uint64_t* bar, uint32_t phase) {
          if (!tc_wait<true>(bar, phase, state)) tc_fail(p.err, state, kDevErrMmaWait);
          __syncwarp();
        };
        // Descriptors are built once a tile; a step adds its 16-byte units to
        // the address, which stays within its 14 bits.  `freed`: the slot
        // whose last reader this product is.
        auto qk = [&](int t, int slot, uint64_t* freed) {
          tc_fence_after();
          if (elect_one()) {
            const uint64_t q = make_sdesc(q_addr + t * Sh::kTileBytes, 16, 1024, 2);
            const uint64_t b = make_sdesc(kv_addr + slot * Sh::kTileBytes, 16, 1024, 2);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              const int off = (k / 4) * 1024 + (k % 4) * 2;
              if (k < k_steps)
                umma_f16(tmem + Sh::kS + t * 128, q + off, b + off, id_qk, k > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[t]);
            if (freed != nullptr) umma_commit(freed);
          }
          __syncwarp();
        };
        // P comes in pieces: the product of one runs while the next one's
        // weights are found.
        uint32_t done[2] = {0, 0};   // key tiles of A and of B so far
        auto pv = [&](int t, int i, int slot, int k0, int k1, uint64_t* freed) {
#pragma unroll
          for (int h = 0; h < kPieces; ++h) {
            prob_meet(t, h, done[t] + static_cast<uint32_t>(i));
            tc_fence_after();
            if (elect_one()) {
              const uint64_t b = make_sdesc(kv_addr + slot * Sh::kTileBytes, 16384, 1024, 2);
              const uint32_t o = tmem + Sh::kO + t * DP, a = tmem + Sh::kS + t * 128;
#pragma unroll
              for (int k = h * (8 / kPieces); k < (h + 1) * (8 / kPieces); ++k)
                if (k >= k0 && k < k1)
                  umma_f16_ta(o, a + k * 8, b + k * 128, id_pv, i > 0 || k > k0 ? 1u : 0u);
              if (h == kPieces - 1) {
                umma_commit(&o_done[t]);
                if (freed != nullptr) umma_commit(freed);
              }
            }
            __syncwarp();
          }
        };
        int k_slot = 0, q_items = 0; // ring slot and phase of the next key tile
        uint32_t k_phase = 0;
        for (int it = 0;; ++it) {
          const TcItem* const d = take(it);
          if (d == nullptr || d->end) break;
          const int n0 = d->n[0], n1 = d->n[1], n = max(n0, n1);
          if (n > 0) {
            const int k_first = v_lo(d->lo, d->start, d->j0) / 16;  // steps of the first key tile
            const int k_last = (v_hi(d->hi_all, d->start, d->j0 + n - 1) + 15) / 16;  // of the last
            wait(&q_full, static_cast<uint32_t>(q_items & 1));
            ++q_items;
            wait(&kv_full[k_slot], k_phase);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int nt = t == 0 ? n0 : n1;
              if (nt == 0) continue;
              if (done[t] > 0) wait(&o_done[t], (done[t] - 1) & 1u);
              qk(t, k_slot, t == 0 && n1 > 0 ? nullptr : &kv_empty[k_slot]);
            }
            if (n == 1) {
              if (elect_one()) umma_commit(&q_empty);
              __syncwarp();
            }
            for (int i = 0; i < n; ++i) {
              int v_slot = k_slot + 1;
              uint32_t v_phase = k_phase;
              if (v_slot == Sh::kSlots) {
                v_slot = 0;
                v_phase ^= 1u;
              }
              k_slot = v_slot + 1;
              k_phase = v_phase;
              if (k_slot == Sh::kSlots) {
                k_slot = 0;
                k_phase ^= 1u;
              }
              wait(&kv_full[v_slot], v_phase);
              if (i + 1 < n) wait(&kv_full[k_slot], k_phase);
              const int k0 = i == 0 ? k_first : 0, k1 = i == n - 1 ? k_last : kKeys / 16;
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                const int nt = t == 0 ? n0 : n1, other = t == 0 ? n1 : 0;
                if (i >= nt) continue;
                pv(t, i, v_slot, k0, k1, i < other ? nullptr : &kv_empty[v_slot]);
                if (i + 1 >= nt) continue;
                // P is read before the next S is written over it.
                wait(&o_done[t], (done[t] + static_cast<uint32_t>(i)) & 1u);
                qk(t, k_slot, i + 1 < other ? nullptr : &kv_empty[k_slot]);
              }
              if (i + 2 == n) {  // the item's last scores are on their way: Q may be replaced
                if (elect_one()) umma_commit(&q_empty);
                __syncwarp();
              }
            }
            done[0] += static_cast<uint32_t>(n0);
            done[1] += static_cast<uint32_t>(n1);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&item_empty[it & 1]);
        }
        // Every MMA completes before tensor memory is freed.
        if (elect_one()) umma_commit(&drain);
        __syncwarp();
        mbar_wait(&drain, 0, nullptr);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------ softmax
    const int t = warp / 4;
    const int row = tid % 128;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t ts = tmem + Sh::kS + t * 128 + lanes, to = tmem + Sh::kO + t * DP + lanes;
    uint32_t done = 0;  // key tiles so far
    bool ok = true;     // until one of this warp's waits has failed
    for (int it = 0;; ++it) {
      const TcItem* const d = take(it);
      if (d == nullptr || d->end) break;
      const int nt = d->n[t];
      // The row's keys [row_beg, row_end), and those that every row of the tile
      // sees, counted from the part's first key tile.
      int row_beg, row_end, all_beg, all_end;
      {
        const int64_t first = d->start + static_cast<int64_t>(d->j0) * kKeys;
        const int64_t place = d->place0 + t * p.tile_tokens;  // of the tile's first token
        auto end_of = [&](int64_t at) {
          const int64_t e = a.causal && at + 1 < d->keys ? at + 1 : d->keys;
          return static_cast<int>(e > first ? e - first : 0);
        };
        auto beg_of = [&](int64_t at) {
          const int64_t b = a.window > 0 ? at - a.window + 1 : 0;
          return static_cast<int>(b > first ? b - first : 0);
        };
        const int tok = row / p.group;
        row_end = end_of(place + tok);
        row_beg = beg_of(place + tok);
        all_end = end_of(place);
        all_beg = beg_of(place + d->tokens[t] - 1);
      }
      float m = -INFINITY, l = 0.0f;
      for (int i = 0; i < nt; ++i) {
        const int kb = i * kKeys;
        const uint32_t n = done + static_cast<uint32_t>(i);
        if (ok && !tc_wait(&s_full[t], n & 1u, state)) {
          tc_fail(p.err, state, kDevErrEpiWait);
          ok = false;
        }
        ok = __all_sync(~0u, ok);
        if (!ok) {
#pragma unroll
          for (int h = 0; h < kPieces; ++h) prob_meet(t, h, n);
          continue;
        }
        tc_fence_after();
        uint32_t s[kKeys];
        tmem_ld128(ts, s);
        const bool edge = kb + kKeys > all_end || kb < all_beg;
        if (edge) {
          const int end = row_end - kb, beg = row_beg - kb;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t seen = low_bits(end - 32 * c) & ~low_bits(beg - 32 * c);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if ((seen >> x & 1u) == 0) s[32 * c + x] = 0xFF800000u;  // -inf
          }
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t* q = s + 32 * c;
          top[c] = fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
#pragma unroll
          for (int x = 2; x < 32; x += 2)
            top[c] = fmaxf(fmaxf(top[c], __uint_as_float(q[x])), __uint_as_float(q[x + 1]));
        }
        const float m2 = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        const bool grow = (m2 - m) * p.scale_log2 > kGrowLog2;
        if (__any_sync(~0u, grow)) {
          const float f = grow ? ex2((m - m2) * p.scale_log2) : 1.0f;
          if (grow) m = m2;
          l *= f;
          if (i > 0) {
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(to + c * 32, o);
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st32(to + c * 32, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m * p.scale_log2;
        const uint64_t scale2 = f2(p.scale_log2, p.scale_log2), base2 = f2(-base, -base);
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const uint32_t* q = s + 32 * c + 2 * x;
            float e0, e1;
            f2_get(f2_fma(f2(__uint_as_float(q[0]), __uint_as_float(q[1])), scale2, base2), e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            sums[x & 1] = f2_add(sums[x & 1], f2(e0, e1));
            w[x] = pack2<T>(e0, e1);
          }
          tmem_st16(ts + c * 16, w);
          if ((c + 1) % (4 / kPieces) == 0) {
            tmem_wait_st();
            tc_fence_before();
            prob_arrive(t, c / (4 / kPieces), n);
          }
        }
        float sa, sb, sc, sd;
        f2_get(sums[0], sa, sb);
        f2_get(sums[1], sc, sd);
        l += (sa + sb) + (sc + sd);
      }
      done += static_cast<uint32_t>(nt);
      if (nt > 0 && ok) {
        ok = tc_wait(&o_done[t], (done - 1) & 1u, state);
        if (!ok) tc_fail(p.err, state, kDevErrEpiWait);
        __syncwarp();
        tc_fence_after();
      }
      ok = __all_sync(~0u, ok);
      // Read back here so that the loop above does not carry them in registers.
      const volatile TcItem* const v_item = &items[it & 1];
      const int64_t row0 = v_item->row0;
      const int head = v_item->head, pieces = v_item->pieces, first_cta = v_item->first_cta;
      // This CTA's piece: it ends the CTA's share if the item begins here.
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (v_item->j0 == 0 ? 1 : 0);
      const int tk = row / p.group;
      const bool real = tk < v_item->tokens[t];
      const int64_t out_row = row0 + t * p.tile_tokens + tk;
      const int h = head * p.group + (row - tk * p.group);
      float check = 0.0f;  // NaN once an output of the row is not finite
      if (ok) {
        const float f = pieces > 1 ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
        const int64_t at = out_row * a.o_token + h * a.o_head;
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          if (nt > 0) {
            tmem_ld32(to + c * 32, o);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0;
          }
          float v[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(o[x]) * f;
          if (real) {
            if (pieces == 1) {
#pragma unroll
              for (int x = 0; x < 32; x += 16)
                if (c * 32 + x < a.dim) {
                  store16<T>(a, at + c * 32 + x, v + x, c * 32 + x + 16 <= a.dim, p.wide_out);
#pragma unroll
                  for (int y = 0; y < 16; ++y) check = fmaf(v[x + y], 0.0f, check);
                }
            } else {
              float4* dst = p.part_o + (slot * (DP / 4) + c * 8) * 256 + t * 128 + row;
#pragma unroll
              for (int x = 0; x < 8; ++x)
                dst[x * 256] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
            }
          }
        }
        const float ml = m == -INFINITY ? -INFINITY : m * p.scale_log2;
        if (real && pieces > 1) p.part_ml[slot * 256 + t * 128 + row] = make_float2(ml, l);
        if (real && pieces == 1 && a.lse != nullptr)
          a.lse[out_row * a.q_heads + h] =
              l == 0.0f ? -INFINITY : (log2f(l) + ml) * 0.69314718055994531f;
      }
      if (pieces > 1) {
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tid == 0) {
          const unsigned arrived = atomicAdd(p.arrived + first_cta, 1u);
          s_last = arrived + 1 == static_cast<unsigned>(pieces);
          if (s_last) p.arrived[first_cta] = 0;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (s_last) {
          __threadfence();
          // Each thread joins a row: its maximum and sum over the pieces, then
          // its columns, kCols at a time.  A piece without a key that counts
          // (sum 0) has nothing to add.
          auto slot_of = [&](int x) {
            return 2 * static_cast<int64_t>(first_cta + x) + (x == 0 ? 1 : 0);
          };
          const int tt = tid / 128, rr = tid % 128;
          const int jt = rr / p.group;
          if (jt < v_item->tokens[tt]) {
            float mm = -INFINITY, sum = 0.0f;
#pragma unroll 4
            for (int x = 0; x < pieces; ++x) {
              const float2 ml = __ldcg(p.part_ml + slot_of(x) * 256 + tid);
              const float top = fmaxf(mm, ml.x);
              const float bs = top == -INFINITY ? 0.0f : top;
              sum = sum * ex2(mm - bs) + ml.y * ex2(ml.x - bs);
              mm = top;
            }
            const float bs = mm == -INFINITY ? 0.0f : mm;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int64_t orow = row0 + tt * p.tile_tokens + jt;
            const int oh = head * p.group + (rr - jt * p.group);
            const int64_t at = orow * a.o_token + oh * a.o_head;
            constexpr int kCols = 32;
#pragma unroll 1
            for (int col = 0; col < DP; col += kCols) {
              float acc[kCols];
#pragma unroll
              for (int y = 0; y < kCols; ++y) acc[y] = 0.0f;
#pragma unroll 4
              for (int x = 0; x < pieces; ++x) {
                const float2 ml = __ldcg(p.part_ml + slot_of(x) * 256 + tid);
                const float f = ex2(ml.x - bs);
                float4 v[kCols / 4];
#pragma unroll
                for (int y = 0; y < kCols / 4; ++y)
                  v[y] = __ldcg(p.part_o + (slot_of(x) * (DP / 4) + col / 4 + y) * 256 + tid);
                if (ml.y != 0.0f)
#pragma unroll
                  for (int y = 0; y < kCols / 4; ++y) {
                    acc[4 * y] = fmaf(v[y].x, f, acc[4 * y]);
                    acc[4 * y + 1] = fmaf(v[y].y, f, acc[4 * y + 1]);
                    acc[4 * y + 2] = fmaf(v[y].z, f, acc[4 * y + 2]);
                    acc[4 * y + 3] = fmaf(v[y].w, f, acc[4 * y + 3]);
                  }
              }
#pragma unroll
              for (int y = 0; y < kCols; ++y) acc[y] *= inv;
#pragma unroll
              for (int y = 0; y < kCols; y += 16)
                if (col + y < a.dim) {
                  store16<T>(a, at + col + y, acc + y, col + y + 16 <= a.dim, p.wide_out);
#pragma unroll
                  for (int z = 0; z < 16; ++z) check = fmaf(acc[y + z], 0.0f, check);
                }
            }
            if (a.lse != nullptr)
              a.lse[orow * a.q_heads + oh] =
                  sum == 0.0f ? -INFINITY : (log2f(sum) + bs) * 0.69314718055994531f;
          }
        }
      }
      const uint32_t bad = __ballot_sync(~0u, check != 0.0f);
      if (bad != 0) {
        AttnRows r;
        const int seq = v_item->seq;
        r.table = a.paged ? a.pages + seq * a.pages_stride : nullptr;
        r.begin = row0 - v_item->place0;  // of packed keys
        r.keys = v_item->keys;
        r.lo = v_item->lo;
        r.hi = v_item->hi_all;
        r.row0 = row0 + t * p.tile_tokens;
        r.place0 = v_item->place0 + t * p.tile_tokens;
        r.head = head;
        r.group = p.group;
        r.first = (warp % 4) * 32;
        if (lane == 0) atomicAdd(state, kRowsAgain);
        __syncwarp();  // other lanes write these rows again: after this lane's stores
        attn_rows_again<T, DP>(a, r, bad);
        __syncwarp();
        if (lane == 0) atomicAdd(state, -kRowsAgain);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[it & 1]);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kCols);
  }
  // Every CTA has asked for its last item: the last one out leaves the
  // counters as it found them.
  if (tid == 0 && more && atomicAdd(p.done, 1u) + 1 == gridDim.x) {
    *p.next = 0;
    *p.done = 0;
  }
}

template <typename T, int DP>
cudaError_t tc_launch(const TcArgs& p, const CUtensorMap& mq, const CUtensorMap& mk,
                      const CUtensorMap& mv, unsigned grid, cudaStream_t s) {
  using Sh = TcShape<DP>;
  static std::atomic<uint64_t> attr_done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if ((attr_done.load() & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(
        k_attn_tc<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
    if (e != cudaSuccess) return e;
    attr_done.fetch_or(bit);
  }
  k_attn_tc<T, DP><<<grid, kTcThreads, Sh::kSmem, s>>>(mq, mk, mv, p);
  return cudaGetLastError();
}

bool map4(CUtensorMap* m, const void* base, const uint64_t (&dims)[4], const int64_t (&strides)[3],
          const uint32_t (&box)[4]) {
  uint64_t d[4], st[3];
  const uint32_t one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) d[i] = dims[i];
  d[0] *= 2;  // bytes
  // The stride of a dimension of one is never used; any valid one will do.
  for (int i = 0; i < 3; ++i)
    st[i] = dims[i + 1] == 1 ? (dims[0] * 2 + 15) / 16 * 16 : static_cast<uint64_t>(strides[i]) * 2;
  return encode_tensor_map(m, base, 4, d, st, box, one, CU_TENSOR_MAP_SWIZZLE_128B) == CUDA_SUCCESS;
}

int pow2_gcd128(int x) {
  int g = 128;
  while (x % g) g /= 2;
  return g;
}

}  // namespace

// What the tensor maps and tiles cover beyond the vector form: a group of at
// most 128 heads, a positive scale (the running maximum is taken over
// unscaled products), pages of whole 8-row swizzle groups and strides that
// are not 0 (a broadcast view) and below a tensor map's 2^40 bytes.
bool attn_tc_covers(const AttnArgs& a) {
  const int64_t most = int64_t{1} << 39;  // elements of 2 bytes
  const int64_t group = a.q_heads / a.kv_heads;
  if (a.q_token >= most || a.q_head >= most / group || a.kv_token >= most || a.kv_head >= most ||
      a.v_token >= most || a.v_head >= most || a.page_stride >= most)
    return false;
  if (group > 128 || !(a.scale > 0.0f)) return false;
  if (a.paged && (a.page_size % 8 != 0 || a.n_pages == 0)) return false;
  if ((a.tokens > 1 && a.q_token == 0) || (a.q_heads > 1 && a.q_head == 0)) return false;
  if (a.kv_heads > 1 && (a.kv_head == 0 || a.v_head == 0)) return false;
  if (a.paged) {
    if ((a.page_size > 1 && a.kv_token == 0) || (a.n_pages > 1 && a.page_stride == 0)) return false;
  } else if (a.tokens > 1 && (a.kv_token == 0 || a.v_token == 0)) {
    return false;
  }
  return true;
}

cudaError_t launch_attn_tc(const AttnArgs& a, const AttnWork& w, cudaStream_t s) {
  const int dp = a.dim <= 64 ? 64 : 128;
  TcArgs p{};
  p.a = a;
  p.err = w.err;
  p.arrived = w.counters;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.group = a.q_heads / a.kv_heads;
  p.tile_tokens = 128 / p.group;
  p.wide_out = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && (a.o_token | a.o_head) % 16 == 0;
  p.box_keys = a.paged ? pow2_gcd128(a.page_size) : kKeys;

  // Pairs at most: every sequence may end in a part of one.
  const int64_t pair_tokens = 2 * p.tile_tokens;
  int64_t pairs = a.tokens / pair_tokens + a.sequences;
  if (a.paged)
    pairs = std::min(pairs, a.sequences * ((a.max_new + pair_tokens - 1) / pair_tokens));
  p.items = pairs * a.kv_heads;
  if (p.items > 0x7FFFFFFF) return cudaErrorInvalidValue;
  // Fewer than kItemsPerSm items an SM may leave some SMs idle at the end.
  const int64_t most_keys = a.paged ? a.pages_stride * a.page_size : a.tokens;
  int64_t grid = std::min<int64_t>(w.num_sms, kAttnCounters - 2);
  p.shares = p.items < static_cast<int64_t>(kItemsPerSm) * grid &&
             most_keys > kCutTiles * kKeys &&
             most_keys < (1 << 28);  // the count stays within 32 bits
  if (p.shares) {
    grid = std::min(grid, p.items * ((most_keys + kMinShare * kKeys - 1) / (kMinShare * kKeys)));
  } else {
    grid = std::min(grid, p.items);
  }
  p.next = w.counters + kAttnCounters - 2;
  p.done = w.counters + kAttnCounters - 1;
  p.part_o = reinterpret_cast<float4*>(w.base);
  p.part_ml = reinterpret_cast<float2*>(w.base + 2 * grid * 256 * dp * sizeof(float));

  CUtensorMap mq, mk, mv;
  const uint64_t dim = a.dim, hkv = a.kv_heads, tok = a.tokens;
  const uint64_t g = p.group;
  bool ok = map4(&mq, a.q, {dim, g, hkv, tok}, {a.q_head, a.q_head * p.group, a.q_token},
                 {128, static_cast<uint32_t>(p.group), 1, static_cast<uint32_t>(p.tile_tokens)});
  const uint32_t box[4] = {128, 1, static_cast<uint32_t>(p.box_keys), 1};
  if (a.paged) {
    const uint64_t dims[4] = {dim, hkv, static_cast<uint64_t>(a.page_size),
                              static_cast<uint64_t>(a.n_pages)};
    ok = ok && map4(&mk, a.k, dims, {a.kv_head, a.kv_token, a.page_stride}, box) &&
         map4(&mv, a.v, dims, {a.v_head, a.v_token, a.page_stride}, box);
  } else {
    ok = ok && map4(&mk, a.k, {dim, hkv, tok, 1}, {a.kv_head, a.kv_token, 0}, box) &&
         map4(&mv, a.v, {dim, hkv, tok, 1}, {a.v_head, a.v_token, 0}, box);
  }
  if (!ok) return cudaErrorInvalidValue;
  const unsigned n = static_cast<unsigned>(grid);
  if (a.dtype == PSPML_DTYPE_F16)
    return dp == 64 ? tc_launch<__half, 64>(p, mq, mk, mv, n, s)
                    : tc_launch<__half, 128>(p, mq, mk, mv, n, s);
  return dp == 64 ? tc_launch<__nv_bfloat16, 64>(p, mq, mk, mv, n, s)
                  : tc_launch<__nv_bfloat16, 128>(p, mq, mk, mv, n, s);
}

}  // namespace pspml
