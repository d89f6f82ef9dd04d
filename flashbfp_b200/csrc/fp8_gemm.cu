// fp8_gemm.cu — y[m, n] = sum_k x[m, k] w[n, k] + bias[n] for e4m3 operands with a power-of-two
// scale per 128 values of a row (fp8_rows.cu), on tcgen05's block-scaled MMA: the scales enter the
// tensor core, so the fp32 accumulator in tensor memory holds the finished sums.
#include <cuda.h>

#include "common.cuh"
#include "fp8_mma.cuh"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {
using namespace sm100;

struct Fp8Args {
  int64_t m, n;
  int nkb;                 // ceil(k / 128): K blocks
  int kgroups;             // ceil(k / 512): scale tiles of a row group
  const void* bias;
  int bias_dtype;
  void* y;
  int y_dtype;
  int64_t ldy;
  int32_t* err;
  int64_t n_tt;            // token tiles
};

struct Fp8Maps {
  CUtensorMap x, w, xs, ws;
};

// Bounded wait (about a second), giving up early once another role of the CTA has.
__device__ __forceinline__ bool fp8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* err,
                                         int site) {
  if (mbar_try_wait(bar, parity)) return true;
  for (uint32_t it = 0; it < (1u << 16); ++it) {
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if ((it & 15) == 15 && *abort_flag) return false;
  }
  *abort_flag = 1;
  atomicExch(err, site);
  return false;
}

// ---------------------------------------------------------------------------------------
// Few tokens. A CTA takes 128 output features (the MMA's M side: 128 weight rows) x BN tokens
// (its N side) and a contiguous range of the K blocks; the CTAs of a cluster share a tile and
// split its K blocks. Per K block one stage: 128 x 128 weight bytes, BN x 128 token bytes
// (128-byte swizzle) and both scale tiles. Warp 0 loads, warp 1 copies the scales to tensor
// memory and issues four MMAs, warps 2-5 read the sums back (a feature per lane). With a split the CTAs
// leave their fp32 tiles in shared memory and each sums and writes a part of the tile, reading
// the others' through the cluster in rank order (a fixed order: same bits every time).
template <int BN>
struct Few {
  static constexpr int kA = 128 * 128, kB = BN * 128, kSf = 512;
  static constexpr int kStage = kA + kB + 2 * kSf;
  static constexpr int kStages = BN <= 32 ? 5 : BN == 64 ? 4 : 6;
  static constexpr int kThreads = 192;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr uint32_t kTmemCols = kAccCols + 8 * kStages <= 128 ? 128 : 256;
  static constexpr int kData = kStages * kStage;
  static_assert(128 * BN * 4 <= kData, "the fp32 tile reuses the stages");
  static_assert(kAccCols + 8 * kStages <= (int)kTmemCols, "tensor memory budget");
  static constexpr int kPad = 1024;                     // swizzled stages start on 1 KB
  static constexpr size_t kSmem = kData + (2 * kStages + 1) * 8 + 16 + kPad;
};

template <int BN>
__global__ void __launch_bounds__(Few<BN>::kThreads) fp8_few_kernel(const Fp8Args a,
                                                                    const __grid_constant__ Fp8Maps M) {
  using C = Few<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // data stages first (every one a multiple of 1 KB), scale tiles behind each stage's operands
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kData);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  uint32_t splits, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(splits));
  rank = cluster_rank();
  const int64_t tile = blockIdx.x / splits;
  const int64_t n0 = tile / a.n_tt * 128, m0 = tile % a.n_tt * BN;
  const int kb0 = (int)((int64_t)a.nkb * rank / splits), kb1 = (int)((int64_t)a.nkb * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_prologue();

  if (warp == 0) {
    if (elect_one_sync()) {
      prefetch_tmap(&M.w); prefetch_tmap(&M.x); prefetch_tmap(&M.ws); prefetch_tmap(&M.xs);
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = fp8_wait(&empty[s], ph ^ 1, abort_flag, a.err, 20))) break;
        uint8_t* st = smem + (size_t)s * C::kStage;
        mbar_arrive_expect_tx(&full[s], C::kStage);
        tma_2d_g2s(st, &M.w, kb * 128, (int)n0, &full[s]);
        tma_2d_g2s(st + C::kA, &M.x, kb * 128, (int)m0, &full[s]);
        tma_2d_g2s(st + C::kA + C::kB, &M.ws, 0, (int)(n0 / 128 * a.kgroups + kb / 4), &full[s]);
        tma_2d_g2s(st + C::kA + C::kB + C::kSf, &M.xs, 0, (int)(m0 / 128 * a.kgroups + kb / 4), &full[s]);
        ++issued;
        if (++s == C::kStages) { s = 0; ph ^= 1; }
      }
      if (!ok)                                           // copies in flight land before the CTA exits
        for (int j = issued > C::kStages ? issued - C::kStages : 0; j < issued; ++j)
          mbar_wait(&full[j % C::kStages], (uint32_t)(j / C::kStages) & 1, 1u << 20);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t kIdesc = idesc_mxf8(128, BN);
      const uint32_t sbase = smem_u32(smem);
      // tokens start at a multiple of BN inside their 128-row scale tile: 32 rows per column
      const uint32_t col_shift = (uint32_t)(m0 % 128) / 32;
      int s = 0;
      uint32_t ph = 0, acc = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = fp8_wait(&full[s], ph, abort_flag, a.err, 21))) break;
        tc_fence_after();
        const uint32_t st = sbase + s * C::kStage;
        const uint32_t sfa = tmem + C::kAccCols + s * 8, sfb = sfa + 4;
        scales_to_tmem<1>(sfa, smem_desc_scales(st + C::kA + C::kB));
        scales_to_tmem<1>(sfb, smem_desc_scales(st + C::kA + C::kB + C::kSf));
        const uint64_t da = smem_desc_sw128(st, 1024), db = smem_desc_sw128(st + C::kA, 1024);
        const uint32_t id = idesc_mxf8_id(kIdesc, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) {                    // 32 values = 32 bytes per step
          mma_mxf8<1>(tmem, da + 2 * k, db + 2 * k, id, sfa, sfb + col_shift, acc);
          acc = 1;
        }
        if (kb + C::kStages < kb1) mma_commit(&empty[s]);   // only where the producer waits for it
        if (++s == C::kStages) { s = 0; ph ^= 1; }
      }
      mma_commit(done);
      if (!ok) mbar_wait(done, 0, 1u << 22);             // MMAs in flight end before their memory goes
    }
    __syncwarp();
  } else if (__all_sync(0xffffffffu, fp8_wait(done, 0, abort_flag, a.err, 22))) {
    tc_fence_after();
    const int q4 = warp & 3, row = q4 * 32 + lane;       // tensor-memory lane = feature n0 + row
    const uint32_t taddr = tmem + ((uint32_t)(q4 * 32) << 16);
    const int ntok = (int)(a.m - m0 < BN ? a.m - m0 : BN);
    const bool store = n0 + row < a.n;
    const float bv = (a.bias && store && splits == 1) ? load_as_float(a.bias, a.bias_dtype, n0 + row) : 0.f;
    float* part = reinterpret_cast<float*>(smem);
    for (int c0 = 0; c0 < ntok; c0 += 16) {
      float v[16];
      if (kb1 > kb0) {
        tmem_ld_32x32b_x16(taddr + c0, v);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int tok = c0 + j;
        if (splits > 1) part[tok * 128 + row] = v[j];    // tok < BN always
        else if (store && tok < ntok)
          store_from_float(a.y, a.y_dtype, (m0 + tok) * a.ldy + n0 + row, v[j] + bv);
      }
    }
  }

  tc_fence_before();
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    const int ntok = (int)(a.m - m0 < BN ? a.m - m0 : BN);
    const uint32_t sbase = smem_u32(smem);
    for (int i = (int)(rank * C::kThreads + threadIdx.x); i < ntok * 128; i += (int)splits * C::kThreads) {
      const int64_t tok = m0 + (i >> 7), feat = n0 + (i & 127);
      float v = 0.f;
      for (uint32_t r = 0; r < splits; ++r) v += ld_shared_cluster(map_shared(sbase + i * 4, r));
      if (feat < a.n) {
        if (a.bias) v += load_as_float(a.bias, a.bias_dtype, feat);
        store_from_float(a.y, a.y_dtype, tok * a.ldy + feat, v);
      }
    }
    __syncwarp();
    cluster_sync();                                      // the tiles stay until every CTA has read them
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int BN>
int launch_few(const Fp8Args& a, const Fp8Maps& M, int dev, int splits, cudaStream_t st) {
  using C = Few<BN>;
  static bool attr_set[64] = {false};
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(fp8_few_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)C::kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t grid = (a.n + 127) / 128 * a.n_tt * splits;
  FBFP_CHECK_ARG(grid < ((int64_t)1 << 31), "too many output tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FBFP_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_few_kernel<BN>, a, M));
  FBFP_LAUNCH_CHECK("fp8_few_kernel");
  return FBFP_OK;
}

// ---------------------------------------------------------------------------------------
// Many tokens. Persistent CTA pairs (cta_group::2): a pair takes tiles of 256 tokens x BN features,
// tokens on the MMA's M side (128 per CTA), features on its N side (half of the weight rows in each
// CTA's shared memory), so that each SM loads 128 + BN / 2 rows of 128 bytes per K block for
// 128 x BN x 128 multiply-adds. Scale tiles are loaded once per 512 values of K, with the stage of
// the group's first K block, and copied to one of kSfSlots slots of tensor memory; a slot is
// written again only when MMAs of at least kStages later K blocks (or of a drained accumulator)
// are due, so the MMAs that read it have completed. A tile starts on a whole scale tile (features
// in steps of 128), which keeps the scales' tensor-memory addresses on multiples of 4 columns.
template <int BN>
struct Many {
  static constexpr int kHalfN = BN / 2;
  static constexpr int kChunks = BN / 128;                       // scale tiles of the features
  static constexpr int kA = 128 * 128, kB = kHalfN * 128, kSf = 512 * (1 + kChunks);
  static constexpr int kStage = kA + kB + 2048;
  static constexpr int kStages = 6;
  static constexpr int kBufs = BN == 256 ? 1 : 2;                // accumulators
  static constexpr int kSfCols = 4 * (1 + kChunks), kSfSlots = 4;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (4 + kEpiWarps);
  static constexpr uint32_t kTmemCols = 512, kSfCol0 = kBufs * BN;
  static constexpr int kData = kStages * kStage;
  static constexpr int kBars = 2 * kStages + 2 + 2 + 1;
  static constexpr size_t kSmem = kData + kBars * 8 + 16 + 1024;
  static_assert(BN % 128 == 0 && kSf <= 2048, "features in whole scale tiles");
  static_assert(kSfCol0 + kSfSlots * kSfCols <= (int)kTmemCols, "tensor memory budget");
  static_assert(kSmem <= 232448, "shared memory budget");
};

struct ManyShared {
  volatile int* abort_flag;
  int32_t* err;
};

__device__ __forceinline__ bool many_wait(uint64_t* bar, uint32_t parity, const ManyShared& S, int site) {
  for (uint32_t it = 0; it < (1u << 16); ++it) {
    if (mbar_try_wait_cluster(bar, parity, 20000u)) return true;
    if ((it & 15) == 15 && *S.abort_flag) return false;
  }
  *S.abort_flag = 1;
  atomicExch(S.err, site);
  return false;
}

// 32 consecutive features of one token. vec: y's rows and base are 32-byte aligned.
__device__ __forceinline__ void store_y32(const Fp8Args& a, int64_t row, int64_t f0, const float (&v)[32], bool vec) {
  if (vec && f0 + 32 <= a.n) {
    if (a.y_dtype == FBFP_F32) {
      float* p = reinterpret_cast<float*>(a.y) + row * a.ldy + f0;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p + 8 * h), "f"(v[8 * h]),
                     "f"(v[8 * h + 1]), "f"(v[8 * h + 2]), "f"(v[8 * h + 3]), "f"(v[8 * h + 4]), "f"(v[8 * h + 5]),
                     "f"(v[8 * h + 6]), "f"(v[8 * h + 7]) : "memory");
    } else {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (a.y_dtype == FBFP_BF16) {
          const __nv_bfloat162 h = __float22bfloat162_rn(make_float2(v[2 * i], v[2 * i + 1]));
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __float22half2_rn(make_float2(v[2 * i], v[2 * i + 1]));
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      uint16_t* p = reinterpret_cast<uint16_t*>(a.y) + row * a.ldy + f0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p + 16 * h), "r"(w[8 * h]),
                     "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]), "r"(w[8 * h + 4]), "r"(w[8 * h + 5]),
                     "r"(w[8 * h + 6]), "r"(w[8 * h + 7]) : "memory");
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (f0 + i < a.n) store_from_float(a.y, a.y_dtype, row * a.ldy + f0 + i, v[i]);
  }
}

template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Many<BN>::kThreads, 1)
fp8_many_kernel(const Fp8Args a, const __grid_constant__ Fp8Maps M) {
  using C = Many<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kData);   // used in CTA 0
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;                               // used in CTA 0
  uint64_t* tail = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 1);
  ManyShared S;
  S.abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  S.err = a.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int64_t tiles = (a.n + BN - 1) / BN * a.n_tt;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * C::kEpiWarps); }
    mbar_init(tail, 1);
    *S.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, C::kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                        // the peer's barriers are ready
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_prologue();

  if (warp == 0) {
    if (elect_one_sync()) {
      prefetch_tmap(&M.w); prefetch_tmap(&M.x); prefetch_tmap(&M.ws); prefetch_tmap(&M.xs);
      const uint32_t sbase = smem_u32(smem);
      int s = 0;
      uint32_t ph = 0;
      int64_t issued = 0;
      bool ok = true;
      for (int64_t t = pair; t < tiles && ok; t += pairs) {
        const int64_t m0 = t % a.n_tt * 256 + 128 * rank, n0 = t / a.n_tt * BN;
        for (int kb = 0; kb < a.nkb; ++kb) {
          if (!(ok = many_wait(&empty[s], ph ^ 1, S, 23))) break;
          const uint32_t st = sbase + (uint32_t)s * C::kStage;
          const uint32_t bar = map_shared(smem_u32(&full[s]), 0);
          const bool sf = (kb & 3) == 0;
          // CTA 0 expects both CTAs' bytes
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2u * (C::kA + C::kB + (sf ? C::kSf : 0)));
          tma_2d_g2s_pair(st, &M.x, kb * 128, (int)m0, bar);
          tma_2d_g2s_pair(st + C::kA, &M.w, kb * 128, (int)(n0 + rank * C::kHalfN), bar);
          if (sf) {
            tma_2d_g2s_pair(st + C::kA + C::kB, &M.xs, 0, (int)(m0 / 128 * a.kgroups + kb / 4), bar);
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)         // tiles past the last one read as zero
              tma_2d_g2s_pair(st + C::kA + C::kB + 512 * (1 + c), &M.ws, 0,
                              (int)((n0 / 128 + c) * a.kgroups + kb / 4), bar);
          }
          ++issued;
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok) {                                         // copies in flight land before the pair exits
        if (rank == 0)
          for (int64_t j = issued > C::kStages ? issued - C::kStages : 0; j < issued; ++j)
            mbar_wait(&full[j % C::kStages], (uint32_t)(j / C::kStages) & 1, 1u << 16);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    if (elect_one_sync()) {
      constexpr uint32_t kIdesc = idesc_mxf8(256, BN);
      const uint32_t sbase = smem_u32(smem);
      const int64_t mine = pair < tiles ? (tiles - pair + pairs - 1) / pairs : 0;
      const int64_t total = mine * a.nkb;
      int64_t it = 0;
      int s = 0, buf = 0, slot = C::kSfSlots - 1;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      for (int64_t t = pair; t < tiles && ok; t += pairs) {
        if (!(ok = many_wait(&acc_empty[buf], aph ^ 1, S, 24))) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        uint32_t acc = 0, sfa = 0;
        for (int kb = 0; kb < a.nkb; ++kb) {
          if (!(ok = many_wait(&full[s], ph, S, 25))) break;
          tc_fence_after();
          const uint32_t st = sbase + (uint32_t)s * C::kStage;
          if ((kb & 3) == 0) {
            slot = slot == C::kSfSlots - 1 ? 0 : slot + 1;
            sfa = tmem + C::kSfCol0 + slot * C::kSfCols;
#pragma unroll
            for (int c = 0; c < 1 + C::kChunks; ++c)
              scales_to_tmem<2>(sfa + 4 * c, smem_desc_scales(st + C::kA + C::kB + 512 * c));
          }
          const uint64_t da = smem_desc_sw128(st, 1024), db = smem_desc_sw128(st + C::kA, 1024);
          const uint32_t id = idesc_mxf8_id(kIdesc, kb & 3);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_mxf8<2>(d, da + 2 * k, db + 2 * k, id, sfa, sfa + 4, acc);
            acc = 1;
          }
          if (it + C::kStages < total) mma_commit_pair(&empty[s]);   // only where the producers wait for it
          ++it;
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        mma_commit_pair(&acc_full[buf]);
        if (++buf == C::kBufs) { buf = 0; aph ^= 1; }
      }
      if (!ok) {                                         // MMAs in flight end before the memory goes
        mma_commit_pair(tail);
        mbar_wait(tail, 0, 1u << 16);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // two warps per lane quarter, half of the columns each: the sums go to registers first, so that
    // the accumulator is free again after the loads
    constexpr int kCols = BN / 2;
    const int q4 = warp & 3, row = q4 * 32 + lane, col0 = ((warp - 4) >> 2) * kCols;
    const bool vec = ((uintptr_t)a.y & 31) == 0 && (a.ldy * (a.y_dtype == FBFP_F32 ? 4 : 2)) % 32 == 0;
    int buf = 0;
    uint32_t ph = 0;
    for (int64_t t = pair; t < tiles; t += pairs) {
      const int64_t tok = t % a.n_tt * 256 + 128 * rank + row, n0 = t / a.n_tt * BN + col0;
      if (!__all_sync(0xffffffffu, many_wait(&acc_full[buf], ph, S, 26))) break;
      tc_fence_after();
      const uint32_t taddr = tmem + buf * BN + col0 + ((uint32_t)(q4 * 32) << 16);
      float v[kCols / 32][32];
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) tmem_ld_32x32b_x32(taddr + 32 * c, v[c]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_shared(smem_u32(&acc_empty[buf]), 0));
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        const int64_t f0 = n0 + 32 * c;
        if (f0 >= a.n) break;                            // whole warps
        if (a.bias) {
          const float b = f0 + lane < a.n ? load_as_float(a.bias, a.bias_dtype, f0 + lane) : 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) v[c][i] += __shfl_sync(0xffffffffu, b, i);
        }
        if (tok < a.m) store_y32(a, tok, f0, v[c], vec);
      }
      if (++buf == C::kBufs) { buf = 0; ph ^= 1; }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();                                        // no CTA leaves while its pair may still reach it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, C::kTmemCols);
  }
}

template <int BN>
int launch_many(const Fp8Args& a, const Fp8Maps& M, int dev, int nsm, cudaStream_t st) {
  using C = Many<BN>;
  static bool attr_set[64] = {false};
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(fp8_many_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)C::kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t tiles = (a.n + BN - 1) / BN * a.n_tt;
  const int64_t pairs = tiles < nsm / 2 ? tiles : nsm / 2;
  FBFP_CUDA_TRY(launch_pdl(fp8_many_kernel<BN>, dim3((unsigned)(2 * pairs)), dim3(C::kThreads), C::kSmem, st, a, M));
  FBFP_LAUNCH_CHECK("fp8_many_kernel");
  return FBFP_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

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
  Fp8Args a;
  a.m = m; a.n = n;
  a.nkb = (int)((k + 127) / 128);
  a.kgroups = (int)((k + 511) / 512);
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.y = y; a.y_dtype = y_dtype; a.ldy = ldy;
  a.err = reinterpret_cast<int32_t*>(workspace);
  int dev = 0;
  FBFP_CUDA_TRY(cudaGetDevice(&dev));
  const int nsm = sm_count(dev);

  constexpr int kManyN = 256;
  const bool many = m > 128;
  const int bn = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;   // token rows of a tile (per CTA)
  a.n_tt = many ? (m + 255) / 256 : (m + bn - 1) / bn;
  const int64_t xt = (m + 127) / 128 * a.kgroups, wt = (n + 127) / 128 * a.kgroups;
  FBFP_CHECK_ARG(xt < ((int64_t)1 << 31) && wt < ((int64_t)1 << 31), "too many scale tiles");
  Fp8Maps M;
  int rc;
  if ((rc = encode_2d(&M.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, x, (uint64_t)k, (uint64_t)m, (uint64_t)ldx, 128,
                      (uint32_t)bn, CU_TENSOR_MAP_SWIZZLE_128B)) != FBFP_OK) return rc;
  if ((rc = encode_2d(&M.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, (uint64_t)k, (uint64_t)n, (uint64_t)ldw, 128,
                      many ? kManyN / 2 : 128, CU_TENSOR_MAP_SWIZZLE_128B)) != FBFP_OK) return rc;
  if ((rc = encode_2d(&M.xs, CU_TENSOR_MAP_DATA_TYPE_UINT32, x_scales, 128, (uint64_t)xt, 512, 128, 1,
                      CU_TENSOR_MAP_SWIZZLE_NONE)) != FBFP_OK) return rc;
  if ((rc = encode_2d(&M.ws, CU_TENSOR_MAP_DATA_TYPE_UINT32, w_scales, 128, (uint64_t)wt, 512, 128, 1,
                      CU_TENSOR_MAP_SWIZZLE_NONE)) != FBFP_OK) return rc;

  const cudaStream_t st = as_stream(stream);
  if (many) return launch_many<kManyN>(a, M, dev, nsm, st);
  // split K over a cluster while that still fills idle SMs (two CTAs fit an SM)
  const int64_t tiles = (n + 127) / 128 * a.n_tt;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= 2 * nsm && a.nkb >= splits * 4) splits *= 2;
  switch (bn) {
    case 16: return launch_few<16>(a, M, dev, splits, st);
    case 32: return launch_few<32>(a, M, dev, splits, st);
    case 64: return launch_few<64>(a, M, dev, splits, st);
    default: return launch_few<128>(a, M, dev, splits, st);
  }
}
