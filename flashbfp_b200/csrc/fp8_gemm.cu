// fp8_gemm.cu — y[m, n] = sum_k x[m, k] w[n, k] + bias[n] for e4m3 operands with a power-of-two
// scale per 128 values of a row (fp8_rows.cu), on tcgen05's block-scaled MMA: the scales enter the
// tensor core, so the fp32 accumulator in tensor memory holds the finished sums.
#include <cuda.h>

#include "common.cuh"
#include "fp8_mma.cuh"
#include "fp8_split.h"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {
using namespace sm100;

struct Fp8Args {
  int64_t m, n;
  uint32_t nkb;            // ceil(k / 128): K blocks
  int kgroups;             // ceil(k / 512): scale tiles of a row group
  const uint8_t *x_scales, *w_scales;
  const void* bias;
  int bias_dtype;
  void* y;
  int64_t ldy;
  int32_t* err;
  uint32_t n_tt;           // token tiles (more than 64 tokens)
  uint32_t tiles;
  int stages;              // depth of the operand ring
};

struct Fp8Maps {
  CUtensorMap x, w, xs, ws;       // the scales' maps: tiles of 128 tokens and more only
};

constexpr int kMaxStages = 8;
// Shared memory a CTA may take so that one or two fit an SM (228 KB, 1 KB of it per CTA reserved).
constexpr int kSmemOne = 232448, kSmemTwo = 115712;

// Where a role of a CTA gave up, and whom it tells.
struct Abort {
  volatile int* flag;
  int32_t* err;
};

// Bounded wait (about a second), giving up early once another role of the CTA has. CLUSTER: other
// CTAs arrive on the barrier too.
template <bool CLUSTER>
__device__ __forceinline__ bool fp8_wait(uint64_t* bar, uint32_t parity, const Abort& A, int site) {
  for (uint32_t it = 0; it < (1u << 16); ++it) {
    if (CLUSTER ? mbar_try_wait_cluster(bar, parity, 20000u) : mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if ((it & 15) == 15 && *A.flag) return false;
  }
  *A.flag = 1;
  atomicExch(A.err, site);
  return false;
}

// After a wait gave up: what is in flight lands before its memory is given up. Each wait has a bound
// of its own again, some 0.3 s times `bounds`.
__device__ __forceinline__ bool settle(uint64_t* bar, uint32_t parity, uint32_t bounds = 1) {
  for (uint32_t it = 0; it < (bounds << 14); ++it)
    if (mbar_try_wait_cluster(bar, parity, 20000u)) return true;
  return false;
}
// The last loads into the stages, of `issued`.
__device__ __forceinline__ void settle_loads(uint64_t* full, int64_t issued, int stages) {
  for (int64_t j = issued > stages ? issued - stages : 0; j < issued; ++j)
    settle(&full[j % stages], (uint32_t)(j / stages) & 1);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __float22bfloat162_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __float22half2_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void round_to(float v, float& o) { o = v; }
__device__ __forceinline__ void round_to(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void round_to(float v, __half& o) { o = __float2half_rn(v); }

// Four consecutive features at p; n of them exist; vec: all four, and p is aligned for one store.
template <typename T>
__device__ __forceinline__ void store4(T* p, int n, const float4& v, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(p) = v;
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, p), pack2(v.z, v.w, p));
  } else {
    if (n > 0) round_to(v.x, p[0]);
    if (n > 1) round_to(v.y, p[1]);
    if (n > 2) round_to(v.z, p[2]);
    if (n > 3) round_to(v.w, p[3]);
  }
}

// ---------------------------------------------------------------------------------------
// Few tokens (up to 64). A CTA takes 128 output features (the MMA's M side: 128 weight rows) x the
// tokens (its N side, BN of them, zeros past the last) and a contiguous range of the K blocks; the
// CTAs of a cluster (up to 8) share a tile and split its K blocks. Per K block one stage: 128 x 128
// weight bytes, BN x 128 token bytes (128-byte swizzle) and both scale tiles. Warp 0 loads, warp 1
// copies the scales to tensor memory and issues four MMAs, warps 2-5 read the sums back (a feature
// per lane) into shared memory. With a split each CTA owns some of the tile's tokens: the others store their fp32
// partial sums straight into its shared memory, and it adds them in rank order (a fixed order: same
// bits every time). Bound by the weights' bytes, and by some 3.4 us of launch, first bytes and
// drain. Measured, in a graph over more weights than L2 holds: 16 x 30720 x 3840 21.9 us
// (5.5 TB/s), 64 x 30720 x 3840 24.2 us (5.1 TB/s), 64 x 8192 x 28672 41.9 us (5.6 TB/s), 1 x 8192
// x 3840 8.4 us, 1 x 3840 x 4096 6.1 us.
template <int BN>
struct Few {
  static constexpr int kA = 128 * 128, kB = BN * 128, kSf = 512;
  static constexpr int kStage = kA + kB + 2 * kSf;
  static constexpr int kSums = (BN + 8) * 512;          // partial sums of the tokens a CTA owns
  static constexpr int kThreads = 192;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr uint32_t kTmemCols = 128;
  static constexpr int kBars = (2 * kMaxStages + 2) * 8 + 16;
  static constexpr int kFixed = kBars + 1024;           // stages start on 1 KB
  static_assert(kStage % 1024 == 0, "swizzled stages start on 1 KB");
  static_assert(kSums <= 3 * kStage, "unsplit, the sums take the place of the stages (at least 3)");
  static_assert(kAccCols + 8 * kMaxStages <= (int)kTmemCols, "tensor memory budget");
};

// After a wait gave up, once every role has ended. (Out of line: inlined, it costs a one-token call 0.1 us.)
__device__ __noinline__ void settle_few(uint64_t* full, uint64_t* done, int64_t issued, int stages) {
  settle_loads(full, issued, stages);
  settle(done, 0);                                       // the MMAs
}

template <int BN, typename T>
__global__ void __launch_bounds__(Few<BN>::kThreads) fp8_few_kernel(const Fp8Args a,
                                                                    const __grid_constant__ Fp8Maps M) {
  using C = Few<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint32_t splits, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(splits));
  rank = cluster_rank();
  const int stages = a.stages;
  // [rank][owned token][feature]: behind the stages, or in their place (one CTA: the MMAs are done)
  float* sums = reinterpret_cast<float*>(smem + (splits > 1 ? stages * C::kStage : 0));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * C::kStage + (splits > 1 ? C::kSums : 0));
  uint64_t* empty = full + kMaxStages;
  uint64_t* done = empty + kMaxStages;
  int64_t* issued_loads = reinterpret_cast<int64_t*>(done + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(issued_loads + 1);
  const Abort A{reinterpret_cast<volatile int*>(tmem_slot + 1), a.err};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int64_t n0 = (int64_t)(blockIdx.x / splits) * 128;
  const int kb0 = (int)(a.nkb * rank / splits), kb1 = (int)(a.nkb * (rank + 1) / splits);   // nkb < 2^24
  const int ntok = (int)a.m;                             // <= BN
  const int own = (int)((ntok + splits - 1) / splits);   // tokens a CTA of the cluster owns
  const int t1 = min(own, ntok - (int)rank * own);       // this one (none: <= 0)

  if (warp == 0 && elect_one_sync()) {
    // the first weights on their way to L2 while the previous kernel of the stream ends
    prefetch_tmap(&M.w); prefetch_tmap(&M.x);
    for (int kb = kb0; kb < kb1 && kb < kb0 + stages; ++kb) tma_2d_prefetch(&M.w, kb * 128, (int)n0);
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    *A.flag = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (splits > 1) cluster_arrive();                      // "this CTA runs": waited for below
  pdl_prologue();

  if (warp == 0) {
    if (elect_one_sync()) {
      int s = 0, kb = kb0;
      uint32_t ph = 0;
      for (; kb < kb1; ++kb) {
        if (!fp8_wait<false>(&empty[s], ph ^ 1, A, 20)) break;
        uint8_t* st = smem + (size_t)s * C::kStage;
        mbar_arrive_expect_tx(&full[s], C::kStage);
        tma_2d_g2s(st, &M.w, kb * 128, (int)n0, &full[s]);
        tma_2d_g2s(st + C::kA, &M.x, kb * 128, 0, &full[s]);
        bulk_g2s(st + C::kA + C::kB, a.w_scales + (n0 / 128 * a.kgroups + kb / 4) * C::kSf, C::kSf, &full[s]);
        bulk_g2s(st + C::kA + C::kB + C::kSf, a.x_scales + (int64_t)(kb / 4) * C::kSf, C::kSf, &full[s]);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      *issued_loads = kb - kb0;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t kIdesc = idesc_mxf8(128, BN);
      const uint32_t sbase = smem_u32(smem);
      int s = 0;
      uint32_t ph = 0, acc = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!fp8_wait<false>(&full[s], ph, A, 21)) break;
        tc_fence_after();
        const uint32_t st = sbase + s * C::kStage;
        const uint32_t sfa = tmem + C::kAccCols + s * 8, sfb = sfa + 4;
        scales_to_tmem<1>(sfa, smem_desc_scales(st + C::kA + C::kB));
        scales_to_tmem<1>(sfb, smem_desc_scales(st + C::kA + C::kB + C::kSf));
        const uint64_t da = smem_desc_sw128(st, 1024), db = smem_desc_sw128(st + C::kA, 1024);
        const uint32_t id = idesc_mxf8_id(kIdesc, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) {                    // 32 values = 32 bytes per step
          mma_mxf8<1>(tmem, da + 2 * k, db + 2 * k, id, sfa, sfb, acc);
          acc = 1;
        }
        if (kb + stages < kb1) mma_commit(&empty[s]);    // only where the producer waits for it
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      mma_commit(done);
    }
    __syncwarp();
  }
  if (splits > 1) cluster_wait();                        // every CTA of the cluster runs
  if (warp >= 2 && __all_sync(0xffffffffu, fp8_wait<false>(done, 0, A, 22))) {
    tc_fence_after();
    const int q4 = warp & 3, row = q4 * 32 + lane;       // tensor-memory lane = feature n0 + row
    const uint32_t taddr = tmem + ((uint32_t)(q4 * 32) << 16);
    const uint32_t slot = smem_u32(sums + rank * own * 128 + row);
    // owner by owner, 16 tokens at a time (columns past the accumulator's are not used)
#pragma unroll 1
    for (int o = 0; o < (int)splits; ++o) {
      const int t0 = o * own, cnt = min(own, ntok - t0);
      const uint32_t dst = splits > 1 ? map_shared(slot, o) : slot;
#pragma unroll 1
      for (int c = 0; c < cnt; c += 16) {
        float v[16];
        tmem_ld_32x32b_x16(taddr + t0 + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < cnt) st_shared_cluster(dst + (c + j) * 512, v[j]);
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (splits > 1) {                                      // every partial sum has landed
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  // a warp per owned token, 4 features per lane
  const int f = lane * 4, nf = (int)(a.n - n0 - f < 4 ? a.n - n0 - f : 4);
  const bool vec = n0 + 128 <= a.n && a.ldy % 4 == 0 && ((uintptr_t)a.y & 15) == 0;
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < nf) bias[i] = load_as_float(a.bias, a.bias_dtype, n0 + f + i);
  T* y = reinterpret_cast<T*>(a.y) + (int64_t)((int)rank * own) * a.ldy + n0 + f;
#pragma unroll 1
  for (int t = warp; t < t1; t += C::kThreads / 32) {
    float4 p = make_float4(bias[0], bias[1], bias[2], bias[3]);
    const float* from = sums + t * 128 + f;
#pragma unroll 4
    for (int r = 0; r < (int)splits; ++r) {
      const float4 q = *reinterpret_cast<const float4*>(from + r * own * 128);
      p.x += q.x; p.y += q.y; p.z += q.z; p.w += q.w;
    }
    store4(y + t * a.ldy, nf, p, vec);
  }
  if (warp == 2) {
    if (*A.flag) {
      settle_few(full, done, *issued_loads, stages);
      __syncwarp();
    }
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------
// Many tokens (more than 64): tokens on the MMA's M side. CG = 1: a CTA takes tiles of 128 tokens x BN
// features. CG = 2: a CTA pair (cta_group::2) takes tiles of 256 tokens x BN features, with 128
// tokens and half of the weight rows in each CTA's shared memory, so that each SM loads
// 128 + BN / 2 rows of 128 bytes per K block for 128 x BN x 128 multiply-adds. Persistent, or with a
// split: the CTAs (pairs) of a cluster share a tile and split its K blocks.
//
// Measured, in a graph over more weights than L2 holds: 2048 x 30720 x 3840 169 to 176
// us in bursts (2.75 to 2.86 PFLOP/s; 202 us at the power limit), 4096 x 8192 x 28672 664 us (2.90
// PFLOP/s), 512 x 8192 x 3840 16.4 us, 128 x 30720 x 3840 26.4 us, 128 x 3840 x 15360 16.5 us (3.8 TB/s). Bound by the
// operand rows an SM can take in, about 60 bytes a cycle: 585 cycles for the 512 of a pair's
// 256-wide K block.
//
// A tile's features are one or two halves of 128, an MMA and an accumulator each; the accumulators
// are a ring of two (BN = 128) or three (BN = 256). So the next tile's first half starts at once
// where the last tile's MMAs end, and its second half follows, up to four K blocks behind, when
// the epilogue has drained the last tile's first half: with one 256-wide accumulator the tensor
// core waited about 2100 of 19700 cycles per tile of 3840 deep.
//
// Scale tiles are loaded once per 512 values of K, with the stage of the group's first K block, and
// copied to one of four slots of tensor memory in turn. A slot is written again 10 or more K
// blocks later where a tile has more than 8 (more than the stages in flight), else at least two
// tiles later (whose accumulators had to be drained first): either way the MMAs that read it
// have completed. A tile starts on a whole scale tile (features in steps of 128), which keeps the
// scales' tensor-memory addresses on multiples of 4 columns.
//
// Epilogue: eight warps, each with 32 tokens (a lane quarter; a token per lane) x 64 features of a
// half. The sums go to registers first, so that the accumulator is free again after the
// loads. With a split every block of 32 tokens x 32 features has an owner among the cluster's CTAs:
// the others store their sums into its shared memory (a warp's store is 512 bytes in a row: 16
// bytes a lane), and it adds them to its own in rank order, once all of them have landed (fp8_split.h).
// Owners are spread so that four warps of every CTA have a block (split four ways) or two (eight
// ways: two warps with one).
template <int CG, int BN>
struct Many {
  static constexpr int kHalves = BN / 128, kRing = kHalves + 1;
  static constexpr int kRowsB = 128 / CG;                        // weight rows of a half in this CTA
  static constexpr int kA = 128 * 128, kHalfB = kRowsB * 128, kB = kHalves * kHalfB, kSf = 512 * (1 + kHalves);
  static constexpr int kStage = kA + kB + (kSf + 1023) / 1024 * 1024;
  static constexpr int kSfCols = 4 * (1 + kHalves), kSfSlots = 4;
  static constexpr uint32_t kSfCol0 = kRing * 128, kTmemCols = 512;
  static constexpr int kEpiWarps = 8, kThreads = 32 * (4 + kEpiWarps);
  static constexpr int kTurn = 32 * 17 * 4;                      // a warp's 32 x 16 words, rows 17 apart
  static constexpr int kTurns = kEpiWarps * kTurn;
  static constexpr int kBlock = 32 * 32 * 4;                     // [feature / 4][token][4]
  static constexpr int kSums = 14 * kBlock;                      // 16 / S blocks from S - 1 CTAs, S 2, 4 or 8
  static constexpr int kBars = (2 * kMaxStages + 2 * kRing + 6) * 8 + 16;
  static constexpr int kFixed = kBars + 1024;                    // stages start on 1 KB
  static_assert(BN % 128 == 0 && kStage % 1024 == 0 && kTurn % 16 == 0 && kBlock % 16 == 0, "alignment");
  static_assert(kSfCol0 + kSfSlots * kSfCols <= kTmemCols, "tensor memory budget");
};

// One warp: 32 consecutive features, the first f0, of 32 consecutive tokens, one per lane (the
// first tok0; tokens from a.m on are not stored). vec, the bytes that y's base and rows are
// aligned to: at 32 each lane stores whole sectors of its row, at 16 halves of them; else the
// values turn through shared memory (`turn`) and the lanes store along the rows.
template <typename T>
__device__ __forceinline__ void store_y32(const Fp8Args& a, int64_t tok0, int64_t f0, const float (&v)[32], int vec,
                                          uint32_t* turn) {
  const int lane = threadIdx.x & 31;
  const int64_t row = tok0 + lane;
  const int rows = a.m - tok0 < 32 ? (int)(a.m - tok0) : 32;
  T* y = reinterpret_cast<T*>(a.y);
  if constexpr (sizeof(T) == 4) {
    if (vec && f0 + 32 <= a.n) {
      if (row >= a.m) return;
      T* p = y + row * a.ldy + f0;
      if (vec == 16) {
#pragma unroll
        for (int h = 0; h < 8; ++h)
          reinterpret_cast<float4*>(p)[h] = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
        return;
      }
#pragma unroll
      for (int h = 0; h < 4; ++h)
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p + 8 * h), "f"(v[8 * h]),
                     "f"(v[8 * h + 1]), "f"(v[8 * h + 2]), "f"(v[8 * h + 3]), "f"(v[8 * h + 4]), "f"(v[8 * h + 5]),
                     "f"(v[8 * h + 6]), "f"(v[8 * h + 7]) : "memory");
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {                        // 16 columns at a time, two rows per store
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) turn[lane * 17 + i] = __float_as_uint(v[16 * h + i]);
      __syncwarp();
      const int64_t f = f0 + 16 * h + (lane & 15);
      const int r1 = f < a.n ? rows : 0;
      T* p = y + (tok0 + (lane >> 4)) * a.ldy + f;
      T q[16];                                           // all loads, then all stores: twice as fast as in turn
#pragma unroll
      for (int r = 0; r < 16; ++r) q[r] = __uint_as_float(turn[(2 * r + (lane >> 4)) * 17 + (lane & 15)]);
#pragma unroll
      for (int r = 0; r < 16; ++r, p += 2 * a.ldy)
        if (2 * r + (lane >> 4) < r1) *p = q[r];
    }
  } else {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], y);
    if (vec && f0 + 32 <= a.n) {
      if (row >= a.m) return;
      T* p = y + row * a.ldy + f0;
      if (vec == 16) {
#pragma unroll
        for (int h = 0; h < 4; ++h)
          reinterpret_cast<uint4*>(p)[h] = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
        return;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p + 16 * h), "r"(w[8 * h]),
                     "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]), "r"(w[8 * h + 4]), "r"(w[8 * h + 5]),
                     "r"(w[8 * h + 6]), "r"(w[8 * h + 7]) : "memory");
      return;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) turn[lane * 17 + i] = w[i];
    __syncwarp();
    const int r1 = f0 + lane < a.n ? rows : 0;
    T* p = y + tok0 * a.ldy + f0 + lane;
    T q[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) q[r] = reinterpret_cast<const T*>(turn + r * 17)[lane];
#pragma unroll
    for (int r = 0; r < 32; ++r, p += a.ldy)
      if (r < r1) *p = q[r];
  }
}

template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar, uint16_t pair_mask) {
  if constexpr (CG == 1) mma_commit(bar);
  else mma_commit_pair(bar, pair_mask);
}
template <int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 1) tma_2d_g2s(dst, map, x, y, bar);
  else tma_2d_g2s_pair(dst, map, x, y, bar);
}

// After a wait gave up, one thread of the CTA, once every role has ended: the loads, the MMAs and the
// other CTAs' sums in flight are waited for. A pair's loads complete on its first CTA's barriers,
// which expect both CTAs' bytes from the first CTA's own load on: the second says how many loads it
// issued, the first makes up the difference where one got further (loads_owed) and lets the second
// go in the end. No barrier of the cluster: every wait is bounded.
template <int CG, int BN>
__device__ __noinline__ void settle_many(uint64_t* full, uint64_t* rest, volatile int64_t* issued, int stages, int kb0,
                                         int kb1, int64_t tiles) {
  using C = Many<CG, BN>;
  uint64_t *told = rest + 1, *landed = rest + 2, *acc_full = full + 2 * kMaxStages;
  const uint32_t rank = cluster_rank(), pr = rank % CG;
  settle(landed, 0);
  if (pr == 1) {
    st_shared_cluster(map_shared(smem_u32((const void*)(issued + 1)), rank - 1), issued[0]);
    mbar_arrive_cluster(map_shared(smem_u32(told), rank - 1));
    settle(rest, 0, kMaxStages + 4);
    return;
  }
  const int64_t mine = issued[0], other = CG == 2 && settle(told, 0, 2) ? issued[1] : mine;
  const int64_t most = mine > other ? mine : other;
  for (int64_t j = mine < other ? mine : other; j < most; ++j) {
    const int kb = kb0 + (int)(j % (kb1 - kb0));
    const uint32_t bytes = C::kA + C::kB + ((kb & 3) == 0 || kb == kb0 ? C::kSf : 0);   // of one CTA
    if (loads_owed(j, mine, other) > 0) mbar_arrive_expect_tx(&full[j % stages], bytes);
    else mbar_complete_tx(&full[j % stages], bytes);
  }
  settle_loads(full, most, stages);
  // the MMAs of whole tiles (a role that gave up has waited for its own)
  const int64_t halves = tiles * C::kHalves;
  for (int64_t h = halves > C::kRing ? halves - C::kRing : 0; h < halves; ++h)
    settle(&acc_full[h % C::kRing], (uint32_t)(h / C::kRing) & 1);
  if constexpr (CG == 2) mbar_arrive_cluster(map_shared(smem_u32(rest), rank + 1));
}

template <int CG, int BN, typename T>
__global__ void __launch_bounds__((Many<CG, BN>::kThreads), 1) fp8_many_kernel(const Fp8Args a, const int splits,
                                                                              const __grid_constant__ Fp8Maps M) {
  using C = Many<CG, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int stages = a.stages;
  // behind the stages: the other CTAs' sums (split) or the epilogue's turning room; a split's
  // epilogue turns in the stages' place, its MMAs being done by then
  uint8_t* sums = smem + stages * C::kStage;
  uint8_t* turns = splits > 1 ? smem : sums;
  uint64_t* full = reinterpret_cast<uint64_t*>(sums + (splits > 1 ? C::kSums : C::kTurns));   // used in a pair's CTA 0
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + C::kRing;                        // used in a pair's CTA 0
  uint64_t* tail = acc_empty + C::kRing;
  uint64_t* rest = tail + 1;
  uint64_t* landed = rest + 2;                                       // told between them (settle_many)
  volatile int64_t* issued_loads = reinterpret_cast<volatile int64_t*>(landed + 1);   // this CTA's, a pair's other's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(landed + 3);
  const Abort A{reinterpret_cast<volatile int*>(tmem_slot + 1), a.err};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), pr = rank % CG, lead = rank - pr;
  const int sp = (int)(rank / CG);                                  // which split of the K blocks
  const uint16_t pair_mask = (uint16_t)(3u << lead);
  const uint32_t team = blockIdx.x / (CG * splits), teams = gridDim.x / (CG * splits);
  const int kb0 = (int)(a.nkb * sp / splits), kb1 = (int)(a.nkb * (sp + 1) / splits);   // nkb < 2^24
  if (warp == 0 && elect_one_sync()) {
    // the first weights on their way to L2 while the previous kernel of the stream ends
    prefetch_tmap(&M.w); prefetch_tmap(&M.x); prefetch_tmap(&M.ws); prefetch_tmap(&M.xs);
    for (int kb = kb0; kb < kb1 && kb < kb0 + stages; ++kb)
      for (int h = 0; h < C::kHalves; ++h)
        tma_2d_prefetch(&M.w, kb * 128, (int)(team / a.n_tt * BN + 128 * h + pr * C::kRowsB));
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < C::kRing; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], CG * C::kEpiWarps); }
    mbar_init(tail, 1);
    mbar_init(rest, 1);
    mbar_init(rest + 1, 1);
    mbar_init(landed, 1);
    *A.flag = 0;
    fence_mbar_init();
    if (splits == 1) {
      mbar_arrive(landed);
    } else {
      const int live = owned_blocks(sp, splits, (int64_t)(team % a.n_tt) * (128 * CG) + 128 * pr,
                                    (int64_t)(team / a.n_tt) * BN, a.m, a.n);
      mbar_arrive_expect_tx(landed, (uint32_t)(live * (splits - 1) * 32 * 32 * 4));
    }
  }
  if (warp == 2) {
    if constexpr (CG == 1) { tmem_alloc(tmem_slot, C::kTmemCols); tmem_relinquish(); }
    else { tmem_alloc_pair(tmem_slot, C::kTmemCols); tmem_relinquish_pair(); }
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (CG == 2) {                               // every CTA of the cluster runs, its barriers are ready
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
    if (splits > 1) cluster_arrive();                    // waited for where the others are needed
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_prologue();

  if (warp == 0) {
    if (elect_one_sync()) {
      const uint32_t sbase = smem_u32(smem);
      int s = 0;
      uint32_t ph = 0;
      int64_t issued = 0;
      bool ok = true;
      for (uint32_t t = team; t < a.tiles && ok; t += teams) {
        const int64_t n0 = (int64_t)(t / a.n_tt) * BN, m0 = (int64_t)(t % a.n_tt) * (128 * CG) + 128 * pr;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = fp8_wait<CG == 2>(&empty[s], ph ^ 1, A, 23))) break;
          const uint32_t st = sbase + (uint32_t)s * C::kStage;
          const uint32_t bar = CG == 1 ? smem_u32(&full[s]) : map_shared(smem_u32(&full[s]), lead);
          const bool sf = (kb & 3) == 0 || kb == kb0;
          // a pair's CTA 0 expects both CTAs' bytes
          if (pr == 0) mbar_arrive_expect_tx(&full[s], CG * (C::kA + C::kB + (sf ? C::kSf : 0)));
          load_tile<CG>(st, &M.x, kb * 128, (int)m0, bar);
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
            load_tile<CG>(st + C::kA + h * C::kHalfB, &M.w, kb * 128, (int)(n0 + 128 * h + pr * C::kRowsB), bar);
          if (sf) {                                      // tiles past the last one read as zero
            load_tile<CG>(st + C::kA + C::kB, &M.xs, 0, (int)(m0 / 128 * a.kgroups + kb / 4), bar);
#pragma unroll
            for (int c = 0; c < C::kHalves; ++c)
              load_tile<CG>(st + C::kA + C::kB + 512 * (1 + c), &M.ws, 0,
                            (int)((n0 / 128 + c) * a.kgroups + kb / 4), bar);
          }
          ++issued;
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
      issued_loads[0] = issued;
      __threadfence_block();                             // the closing barrier may order nothing
    }
    __syncwarp();
  } else if (warp == 1 && pr == 0) {
    if (elect_one_sync()) {
      constexpr uint32_t kIdesc = idesc_mxf8(128 * CG, 128);
      constexpr int kAhead = 4;                          // K blocks of a first half before its second
      const uint32_t sbase = smem_u32(smem);
      const int64_t total = (int64_t)((a.tiles - team + teams - 1) / teams) * (kb1 - kb0);   // team < tiles
      int64_t it = 0;
      int s = 0, slot = C::kSfSlots - 1, ring = 0;
      uint32_t ph = 0, rph = 0, sfa = 0;
      bool ok = true;
      // a half's four MMAs of K block kb (32 values = 32 bytes per step), in stage `stage`
      auto issue = [&](int half, uint32_t acc_slot, int stage, int kb) {
        const uint32_t st = sbase + (uint32_t)stage * C::kStage;
        const uint64_t da = smem_desc_sw128(st, 1024), db = smem_desc_sw128(st + C::kA + half * C::kHalfB, 1024);
        const uint32_t id = idesc_mxf8_id(kIdesc, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_mxf8<CG>(tmem + acc_slot * 128, da + 2 * k, db + 2 * k, id, sfa, sfa + 4 + 4 * half, kb > kb0 || k > 0);
      };
      auto release = [&](int stage) {                    // only where the producers wait for it
        if (it + stages < total) commit<CG>(&empty[stage], pair_mask);
        ++it;
      };
      for (uint32_t t = team; t < a.tiles && ok; t += teams) {
        const uint32_t first = ring, fph = rph;
        if (++ring == C::kRing) { ring = 0; rph ^= 1; }
        const uint32_t second = ring, sph = rph;         // (two halves)
        if (C::kHalves == 2 && ++ring == C::kRing) { ring = 0; rph ^= 1; }
        if (!(ok = fp8_wait<CG == 2>(&acc_empty[first], fph ^ 1, A, 24))) break;
        tc_fence_after();
        bool open = false;                               // the second half's accumulator is free
        int s0 = s;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = fp8_wait<CG == 2>(&full[s], ph, A, 25))) break;
          tc_fence_after();
          if ((kb & 3) == 0 || kb == kb0) {
            const uint32_t st = sbase + (uint32_t)s * C::kStage;
            slot = slot == C::kSfSlots - 1 ? 0 : slot + 1;
            sfa = tmem + C::kSfCol0 + slot * C::kSfCols;
#pragma unroll
            for (int c = 0; c < 1 + C::kHalves; ++c)
              scales_to_tmem<CG>(sfa + 4 * c, smem_desc_scales(st + C::kA + C::kB + 512 * c));
          }
          issue(0, first, s, kb);
          if constexpr (C::kHalves == 1) {
            release(s);
          } else if (open) {
            issue(1, second, s, kb);
            release(s);
          } else {
            // a tile's first blocks share one scale group: kb0 = 0 with two halves, kAhead <= 4
            open = mbar_test(&acc_empty[second], sph ^ 1);
            if (!open && (kb + 1 == kb1 || kb + 1 == kb0 + kAhead)) {
              if (!(ok = fp8_wait<CG == 2>(&acc_empty[second], sph ^ 1, A, 24))) break;
              open = true;
            }
            if (open) {
              tc_fence_after();
              for (int j = kb0; j <= kb; ++j) {
                issue(1, second, s0, j);
                release(s0);
                if (++s0 == stages) s0 = 0;
              }
            }
          }
          if (++s == stages) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        commit<CG>(&acc_full[first], pair_mask);
        if constexpr (C::kHalves == 2) commit<CG>(&acc_full[second], pair_mask);
      }
      if (!ok) {                                         // MMAs in flight end before the memory goes
        commit<CG>(tail, pair_mask);
        mbar_wait(tail, 0, 1u << 16);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q4 = warp & 3, side = (warp - 4) >> 2;
    if (CG == 1 && splits > 1) cluster_wait();           // the owners' barriers are ready
    uint32_t* turn = reinterpret_cast<uint32_t*>(turns + (warp - 4) * C::kTurn);
    const uint64_t bits = (uint64_t)(uintptr_t)a.y | (uint64_t)a.ldy * sizeof(T);
    const int vec = (bits & 31) == 0 ? 32 : (bits & 15) == 0 ? 16 : 0;
    int ring = 0;
    uint32_t ph = 0;
    uint32_t t = team;
    int half = 0;
    int64_t drained = 0;                                 // halves so far, of all
    const int64_t halves = (int64_t)((a.tiles - team + teams - 1) / teams) * C::kHalves;   // team < tiles
#pragma unroll 1
    for (; t < a.tiles; half == C::kHalves - 1 ? (half = 0, t += teams) : ++half) {
      const int64_t tok0 = (int64_t)(t % a.n_tt) * (128 * CG) + 128 * pr + q4 * 32;
      const int64_t n0 = (int64_t)(t / a.n_tt) * BN + 128 * half + 64 * side;
      if (!__all_sync(0xffffffffu, fp8_wait<CG == 2>(&acc_full[ring], ph, A, 26))) break;
      tc_fence_after();
      const uint32_t taddr = tmem + ring * 128 + 64 * side + ((uint32_t)(q4 * 32) << 16);
      float v[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(taddr + 32 * c, v[c]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      // only where an MMA waits for it: a pair's CTA 0 is gone otherwise when the arrival comes
      if (lane == 0 && arrival_awaited(drained++, C::kRing, halves)) {
        if constexpr (CG == 1) mbar_arrive(&acc_empty[ring]);
        else mbar_arrive_cluster(map_shared(smem_u32(&acc_empty[ring]), lead));
      }
      if (++ring == C::kRing) { ring = 0; ph ^= 1; }
      if constexpr (BN == 128) {
        if (splits > 1) {
          // into the owner's room for this block and split
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int owner = block_owner(q4, 2 * side + c, splits);
            if (owner == sp || !block_live(tok0, n0 + 32 * c, a.m, a.n)) continue;
            const int to = owner * CG + pr, from = sp < owner ? sp : sp - 1;
            const int room = block_slot(q4, 2 * side + c, splits) * (splits - 1) + from;
            const uint32_t dst = map_shared(smem_u32(sums) + room * C::kBlock + lane * 16, to);
            const uint32_t bar = map_shared(smem_u32(landed), to);
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              st_async_v4(dst + i * 128, v[c][i], v[c][i + 1], v[c][i + 2], v[c][i + 3], bar);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int64_t f0 = n0 + 32 * c;
        if (!block_live(tok0, f0, a.m, a.n)) break;      // whole warps
        if constexpr (BN == 128) {
          if (splits > 1) {
            if (block_owner(q4, 2 * side + c, splits) != sp) continue;
            if (!__all_sync(0xffffffffu, fp8_wait<true>(landed, 0, A, 27))) break;
            const uint8_t* p = sums + block_slot(q4, 2 * side + c, splits) * (splits - 1) * C::kBlock + lane * 16;
#pragma unroll 1
            for (int r = 0; r < splits - 1; ++r, p += C::kBlock) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 q = *reinterpret_cast<const float4*>(p + i * 128);
                v[c][i] += q.x; v[c][i + 1] += q.y; v[c][i + 2] += q.z; v[c][i + 3] += q.w;
              }
            }
          }
        }
        if (a.bias) {
          const float b = f0 + lane < a.n ? load_as_float(a.bias, a.bias_dtype, f0 + lane) : 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) v[c][i] += __shfl_sync(0xffffffffu, b, i);
        }
        store_y32<T>(a, tok0, f0, v[c], vec, turn);
      }
    }
  }
  __syncwarp();
  if (CG == 1 && splits > 1 && warp < 4) cluster_wait();
  if (*A.flag) {                                         // a wait gave up: the other CTA of a pair is told
    if constexpr (CG == 2) st_shared_cluster(map_shared(smem_u32((const void*)A.flag), rank ^ 1), 1u);
    fence_cluster();                                     // the closing barrier orders nothing by itself
  }
  __syncwarp();
  tc_fence_before();
  // every role of the cluster has ended; no memory is ordered by this: what CTAs send each other is
  // waited for on barriers of its own
  if (CG == 2 || splits > 1) {
    cluster_arrive_relaxed();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 2) {
    if (*A.flag) {                                       // the same in a pair's CTAs from here on
      if (lane == 0)
        settle_many<CG, BN>(full, rest, issued_loads, stages, kb0, kb1, (int64_t)((a.tiles - team + teams - 1) / teams));
      __syncwarp();
    }
    tc_fence_after();
    if constexpr (CG == 1) tmem_dealloc(tmem, C::kTmemCols);
    else tmem_dealloc_pair(tmem, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------
// Launch with programmatic stream serialisation and a cluster of `cluster` CTAs.
template <typename... KArgs, typename... Args>
int launch_cluster(void (*kernel)(KArgs...), int dev, bool (&attr_set)[64], int64_t grid, int cluster, int threads,
                   size_t smem, cudaStream_t st, Args... args) {
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOne));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  FBFP_CHECK_ARG(grid < ((int64_t)1 << 31), "too many output tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FBFP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  FBFP_LAUNCH_CHECK("fp8_linear");
  return FBFP_OK;
}

// How many clusters of `cluster` CTAs run at a time (clusters do not span the SM groups of the chip,
// so the largest leave SMs idle: on 148 SMs, one CTA each, 74 of 2, 33 of 4, 15 of 8).
template <typename... KArgs>
int clusters_at_a_time(void (*kernel)(KArgs...), int dev, int (&known)[64][9], int cluster, int threads, size_t smem) {
  if (dev >= 0 && dev < 64 && known[dev][cluster] > 0) return known[dev][cluster];
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOne);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) n = 1;
  cudaGetLastError();
  if (dev >= 0 && dev < 64) known[dev][cluster] = n;
  return n;
}

// K is split over as large a cluster (up to 8) as leaves every CTA at least 4 K blocks and all tiles
// running at a time: one CTA per SM where these fill 70% of the SMs, else two per SM. A CTA that has
// an SM to itself and more than twice the K blocks of the ring that two leave room for takes the
// larger ring; the others keep the small one, beside which the next kernel's CTAs start. No ring has
// more stages than its CTA has K blocks. Measured, larger / small ring, weights read from HBM: 64 x
// 8192 x 28672 42.6 / 52.4 us, 64 x 3840 x 15360 13.9 / 16.8; read from L2: 1 x 3840 x 4096 5.5 /
// 4.5. One / two per SM: 16 x 18944 x 3840 13.8 / 14.6, 16 x 30720 x 3840 24.9 / 21.2, 32 x 10240 x
// 3840 11.8 / 10.1. In timings of every split of 172 shapes the choice is 1.6% behind the best
// with weights from HBM (11% at worst) and 2.9% with weights from L2 (19%). Occupancy counted one
// CTA per SM for this kernel at 80 to 113 KB of shared memory too, where two do run (296 tiles take
// one round): twice the count is taken for two.
template <int BN, typename T>
int launch_few(Fp8Args a, const Fp8Maps& M, int dev, cudaStream_t st) {
  using C = Few<BN>;
  static bool attr_set[64] = {false};
  static int known[64][9];
  const auto kernel = fp8_few_kernel<BN, T>;
  const int64_t tiles = (a.n + 127) / 128;
  auto clusters = [&](int c) { return (int64_t)clusters_at_a_time(kernel, dev, known, c, C::kThreads, kSmemOne); };
  auto split = [&](int per_sm) {
    for (int c = 8; c > 1; --c)
      if ((int)a.nkb >= 4 * c && tiles <= per_sm * clusters(c)) return c;
    return 1;
  };
  const int64_t sms = clusters(1);
  const int one = split(1);
  const int splits = tiles <= sms && tiles * one * 10 >= sms * 7 ? one : split(2);
  const int extra = splits > 1 ? C::kSums : 0;
  const int blocks = (int)((a.nkb + splits - 1) / splits);
  int stages = (kSmemTwo - C::kFixed - extra) / C::kStage;
  if (tiles <= sms && splits == one && blocks > 2 * stages) stages = (kSmemOne - C::kFixed - extra) / C::kStage;
  if (stages > kMaxStages) stages = kMaxStages;
  if (stages > blocks) stages = blocks < 3 ? 3 : blocks;   // at least 3: the sums' place without a split
  a.stages = stages;
  return launch_cluster(kernel, dev, attr_set, tiles * splits, splits, C::kThreads,
                        (size_t)stages * C::kStage + extra + C::kFixed, st, a, M);
}

template <int CG, int BN, typename T>
int launch_many(Fp8Args a, const Fp8Maps& M, int dev, int teams, int splits, cudaStream_t st) {
  using C = Many<CG, BN>;
  static bool attr_set[64] = {false};
  const int extra = splits > 1 ? C::kSums : C::kTurns;
  const int fit = (kSmemOne - C::kFixed - extra) / C::kStage;
  a.stages = fit < kMaxStages ? fit : kMaxStages;
  return launch_cluster(fp8_many_kernel<CG, BN, T>, dev, attr_set, (int64_t)teams * CG * splits, CG * splits,
                        C::kThreads, (size_t)a.stages * C::kStage + extra + C::kFixed, st, a, splits, M);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

struct Fp8Operands {
  const void *x, *w;
  int64_t k, ldx, ldw;
};

int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t ld, int box) {
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, (uint64_t)k, (uint64_t)rows, (uint64_t)ld, 128,
                   (uint32_t)box, CU_TENSOR_MAP_SWIZZLE_128B);
}
int encode_scales(CUtensorMap* map, const void* base, int64_t tiles) {
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 128, (uint64_t)tiles, 512, 128, 1,
                   CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Which tile and split: the least of an estimate in SM cycles, rounds of tiles x (K blocks x
// cycles per block + 2000 for a tile's fill and drain, 3500 for a pair's) + 5000 for a split's exchange of partial
// sums. Cycles per K block: 128 x BN x 128 multiply-adds take 2 BN, and the operand rows come in
// at about 60 bytes a cycle: measured 520 (one CTA, 128 features; bound by the loads), 768 (256
// features), 500 and 580 (a pair). Measured against the alternatives: 512 tokens x 8192 x 3840
// 16.3 us on 256-wide pair tiles and 18.4 on 128-wide ones, 512 x 3840 x 15360 the other way
// around (40.2 and 31.0 us: 30 and 60 tiles for 74 pairs), 128 x 3840 x 15360 16.1 us split four
// ways, 21.7 two ways, 256 x 3840 x 4096 10.6 split and 11.0 not. Clusters of 8 are for products
// of at most 15 tiles, all that run at a time: 128 x 1920 x 15360 12.2 us, 14.3 split four ways, 100 x
// 1000 x 16000 11.1 and 13.6, 100 x 512 x 8192 7.7 and 9.0; at 4096 deep they are even (0.93 to 1.01
// of the time in 22 shapes of up to 8 tiles) and lose where 12 to 15 tiles leave few SMs idle
// anyway (128 x 1920 x 4096 8.4 and 7.7). One tile more takes a second round: 100 x 2000 x 16000
// (16 tiles) 14.5 us split four ways, 21.2 eight ways.
struct ManyPlan {
  int cg, bn, splits, teams;
  int64_t token_tiles, tiles;
};
ManyPlan plan_many(int64_t m, int64_t n, int nkb, int dev) {
  static int known[64][9];
  const auto kernel = fp8_many_kernel<1, 128, float>;    // one CTA per SM, as all of them
  const int threads = Many<1, 128>::kThreads;
  ManyPlan best{};
  double least = 0;
  for (int cg = 1; cg <= 2; ++cg)
    for (int bn = 128; bn <= 256; bn += 128)
      for (int splits = 1; splits * cg <= 8 && (splits == 1 || (bn == 128 && nkb >= 4 * splits)); splits *= 2) {
        const int64_t tt = (m + 128 * cg - 1) / (128 * cg), tiles = (n + bn - 1) / bn * tt;
        const int64_t slots = clusters_at_a_time(kernel, dev, known, cg * splits, threads, kSmemOne);
        if (splits > 1 && tiles > slots) continue;
        const int64_t rounds = (tiles + slots - 1) / slots;
        const double per_kb = cg == 1 ? (bn == 128 ? 520 : 768) : (bn == 128 ? 500 : 580);
        const double cost = (double)rounds * ((nkb + splits - 1) / splits * per_kb + (cg == 1 ? 2000 : 3500)) +
                            (splits > 1 ? 5000 : 0);
        if (best.cg == 0 || cost < least) {
          least = cost;
          best = ManyPlan{cg, bn, splits, (int)(tiles < slots ? tiles : slots), tt, tiles};
        }
      }
  return best;
}

template <typename T>
int fp8_dispatch(Fp8Args& a, const Fp8Operands& o, int dev, cudaStream_t st) {
  Fp8Maps M;
  int rc;
  if (a.m <= 64) {
    const int bn = a.m <= 16 ? 16 : a.m <= 32 ? 32 : 64;
    if ((rc = encode_rows(&M.x, o.x, a.m, o.k, o.ldx, bn)) != FBFP_OK) return rc;
    if ((rc = encode_rows(&M.w, o.w, a.n, o.k, o.ldw, 128)) != FBFP_OK) return rc;
    return bn == 16   ? launch_few<16, T>(a, M, dev, st)
           : bn == 32 ? launch_few<32, T>(a, M, dev, st)
                      : launch_few<64, T>(a, M, dev, st);
  }
  const ManyPlan p = plan_many(a.m, a.n, (int)a.nkb, dev);
  FBFP_CHECK_ARG(p.tiles < ((int64_t)1 << 31), "too many output tiles");
  a.n_tt = (uint32_t)p.token_tiles;
  a.tiles = (uint32_t)p.tiles;
  if ((rc = encode_rows(&M.x, o.x, a.m, o.k, o.ldx, 128)) != FBFP_OK) return rc;
  if ((rc = encode_rows(&M.w, o.w, a.n, o.k, o.ldw, 128 / p.cg)) != FBFP_OK) return rc;
  if ((rc = encode_scales(&M.xs, a.x_scales, (a.m + 127) / 128 * a.kgroups)) != FBFP_OK) return rc;
  if ((rc = encode_scales(&M.ws, a.w_scales, (a.n + 127) / 128 * a.kgroups)) != FBFP_OK) return rc;
  if (p.cg == 1)
    return p.bn == 128 ? launch_many<1, 128, T>(a, M, dev, p.teams, p.splits, st)
                       : launch_many<1, 256, T>(a, M, dev, p.teams, p.splits, st);
  return p.bn == 128 ? launch_many<2, 128, T>(a, M, dev, p.teams, p.splits, st)
                     : launch_many<2, 256, T>(a, M, dev, p.teams, p.splits, st);
}

}  // namespace
}  // namespace fbfp

using namespace fbfp;

extern "C" int fbfp_fp8_linear(const void* x, int64_t m, int64_t k, int64_t ldx, const void* x_scales, const void* w,
                               int64_t n, int64_t ldw, const void* w_scales, const void* bias, int bias_dtype,
                               void* y, int y_dtype, int64_t ldy, void* workspace, void* stream) {
  FBFP_CHECK_ARG(x && x_scales && w && w_scales && y && workspace, "null pointer");
  FBFP_CHECK_ARG(m >= 1 && m < ((int64_t)1 << 31) - 256 && n >= 1 && n < ((int64_t)1 << 31) - 256 && k >= 1 &&
                     k < ((int64_t)1 << 31) - 256,
                 "bad sizes (m %lld, n %lld, k %lld)", (long long)m, (long long)n, (long long)k);
  FBFP_CHECK_ARG(ldx >= k && ldx % 16 == 0 && ldw >= k && ldw % 16 == 0 && aligned16(x) && aligned16(w),
                 "operands must be 16-byte aligned with rows a multiple of 16 apart (ldx %lld, ldw %lld)",
                 (long long)ldx, (long long)ldw);
  FBFP_CHECK_ARG(aligned16(x_scales) && aligned16(w_scales), "scales must be 16-byte aligned");
  FBFP_CHECK_ARG(ldy >= n, "ldy %lld below n %lld", (long long)ldy, (long long)n);
  FBFP_CHECK_ARG(dtype_ok(y_dtype) && (!bias || dtype_ok(bias_dtype)), "bad y or bias dtype");
  FBFP_CHECK_ARG((uintptr_t)y % dtype_size(y_dtype) == 0 && (!bias || (uintptr_t)bias % dtype_size(bias_dtype) == 0) &&
                     ((uintptr_t)workspace & 3) == 0,
                 "y, bias and workspace must be aligned to their types");
  Fp8Args a;
  a.m = m; a.n = n;
  a.nkb = (uint32_t)((k + 127) / 128);
  a.kgroups = (int)((k + 511) / 512);
  FBFP_CHECK_ARG((m + 127) / 128 * a.kgroups < ((int64_t)1 << 31) && (n + 127) / 128 * a.kgroups < ((int64_t)1 << 31),
                 "too many scale tiles");
  a.x_scales = reinterpret_cast<const uint8_t*>(x_scales);
  a.w_scales = reinterpret_cast<const uint8_t*>(w_scales);
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.y = y; a.ldy = ldy;
  a.err = reinterpret_cast<int32_t*>(workspace);
  const Fp8Operands o{x, w, k, ldx, ldw};
  int dev = 0;
  FBFP_CUDA_TRY(cudaGetDevice(&dev));
  const cudaStream_t st = as_stream(stream);
  return y_dtype == FBFP_BF16  ? fp8_dispatch<__nv_bfloat16>(a, o, dev, st)
         : y_dtype == FBFP_F16 ? fp8_dispatch<__half>(a, o, dev, st)
                               : fp8_dispatch<float>(a, o, dev, st);
}
