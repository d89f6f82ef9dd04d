// fp8_split.h — what the CTAs of a cluster send each other in the block-scaled product: who adds what
// where they share a tile and split its K blocks, and which arrivals are waited for. Plain C++
// beside the kernel (fp8_gemm.cu), so that the rules can be run on the host.
//
// A CTA's 128 tokens x 128 features of sums are 16 blocks of 32 x 32: lane quarter q (tokens), column
// c (features). Each has an owner among the splits: the others store their sums into its shared
// memory, in the order of their rank, and it adds them to its own. A block without a token or
// without a feature has no owner that waits for it, so nothing may be sent for it either: a CTA
// leaves once every byte that is sent to it has landed.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FBFP_HD __host__ __device__ __forceinline__
#else
#define FBFP_HD inline
#endif

namespace fbfp {

// The split whose CTA owns block (q, c) of a split two, four or eight ways, and the block's place
// among that CTA's.
FBFP_HD int block_owner(int q, int c, int splits) {
  return splits == 2 ? c >> 1 : splits == 4 ? c : 2 * c + (q >> 1);
}
FBFP_HD int block_slot(int q, int c, int splits) {
  return splits == 2 ? q * 2 + (c & 1) : splits == 4 ? q : q & 1;
}
// Whether the block whose first token is tok and first feature f has sums to add.
FBFP_HD bool block_live(int64_t tok, int64_t f, int64_t m, int64_t n) { return tok < m && f < n; }
// How many blocks split sp adds of the 128 x 128 that start at token tok and feature f.
FBFP_HD int owned_blocks(int sp, int splits, int64_t tok, int64_t f, int64_t m, int64_t n) {
  int live = 0;
  for (int b = 0; b < 16; ++b)
    live += block_owner(b >> 2, b & 3, splits) == sp && block_live(tok + (b >> 2) * 32, f + (b & 3) * 32, m, n);
  return live;
}

// Whether the MMAs wait for half h (of `halves` that a CTA or pair computes in turn) to be drained: the
// half `ring` later takes its accumulator. An arrival that nobody waits for must not be sent to
// another CTA, which may have left.
FBFP_HD bool arrival_awaited(int64_t h, int ring, int64_t halves) { return h + ring < halves; }

// Loads of a pair complete on its first CTA's barriers: that CTA's own load arrives there and expects
// both CTAs' bytes. After a failure, `mine` loads of the first CTA and `other` of the second having
// been issued, its barrier of load j (j at least the smaller of the two) lacks: an arrival that
// expects the second CTA's bytes (1), or the bytes that the second CTA never sends (-1).
FBFP_HD int loads_owed(int64_t j, int64_t mine, int64_t other) {
  return j >= mine && j < other ? 1 : j < mine && j >= other ? -1 : 0;
}

}  // namespace fbfp
