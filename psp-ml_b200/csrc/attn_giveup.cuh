// attn_giveup.cuh - how the warps of the tensor-core attention kernel
// (attn_tc.cu) stop together once a wait of one of them has run out.
//
// Two of their meetings have no limit of their own: the hardware barriers at
// which the softmax warps hand the weights P to the MMA warp, and those of the
// softmax warps among themselves.  They end because every warp comes to every
// one of them exactly once, whatever its other waits report:
//   * all warps walk the same items.  The loader publishes item after item, and
//     a warp whose wait for the next one runs out closes the book at that item,
//     unless the loader got there first; a single word decides which, so that
//     no warp walks an item that another one has given up;
//   * within an item a warp whose wait failed goes on to all its meetings.  A
//     softmax warp then meets the MMA warp (it waits there) instead of only
//     leaving its arrival, since without the scores' barrier nothing else keeps
//     it from arriving twice in one generation.  What it left before may not
//     have been taken up: odd and even key tiles have barriers of their own, so
//     an arrival left at one tile does not count at the next.
#pragma once

namespace pspml {

// Hardware barrier of piece h of tile t's P at the CTA's n-th key tile for
// tile t: after 0 (the block) and 1 (the softmax warps).
__host__ __device__ constexpr int prob_barrier(int t, int h, unsigned n) {
  return 2 + (2 * t + h) * 2 + static_cast<int>(n & 1u);
}

// The book of items: how many the loader has published, or kItemsClosed.
constexpr int kItemsClosed = -1;

#if defined(__CUDACC__)
// Publishes item `it`; false if the book was closed there.
__device__ __forceinline__ bool item_publish(int* book, int it) {
  __threadfence_block();  // the item's record first
  return atomicCAS(book, it, it + 1) == it;
}
// Gives up on item `it`; false if it has been published after all.
__device__ __forceinline__ bool item_close(int* book, int it) {
  const int was = atomicCAS(book, it, kItemsClosed);
  __threadfence_block();
  return was == it || was == kItemsClosed;
}
#endif

}  // namespace pspml
