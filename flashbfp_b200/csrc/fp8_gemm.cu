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
  const uint8_t *x_scales, *w_scales;
  const void* bias;
  int bias_dtype;
  void* y;
  int y_dtype;
  int64_t ldy;
  int32_t* err;
  int64_t n_tt;            // token tiles
};

struct Fp8Maps {
  CUtensorMap x, w, xs, ws;       // the scales' maps: many tokens only
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

// Four consecutive features (the first is `feat`) at element `at` of y; vec: all four exist and
// the address is aligned for one store.
__device__ __forceinline__ void store4(const Fp8Args& a, int64_t at, int64_t feat, float v0, float v1, float v2,
                                       float v3, bool vec) {
  if (vec) {
    if (a.y_dtype == FBFP_F32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.y) + at) = make_float4(v0, v1, v2, v3);
    } else if (a.y_dtype == FBFP_BF16) {
      const __nv_bfloat162 h[2] = {__float22bfloat162_rn(make_float2(v0, v1)),
                                   __float22bfloat162_rn(make_float2(v2, v3))};
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.y) + at) = *reinterpret_cast<const uint2*>(h);
    } else {
      const __half2 h[2] = {__float22half2_rn(make_float2(v0, v1)), __float22half2_rn(make_float2(v2, v3))};
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.y) + at) = *reinterpret_cast<const uint2*>(h);
    }
  } else {
    const float v[4] = {v0, v1, v2, v3};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (feat + i < a.n) store_from_float(a.y, a.y_dtype, at + i, v[i]);
  }
}

// ---------------------------------------------------------------------------------------
// Few tokens. A CTA takes 128 output features (the MMA's M side: 128 weight rows) x BN tokens
// (its N side) and a contiguous range of the K blocks; the CTAs of a cluster (up to 8) share a tile
// and split its K blocks. Per K block one stage: 128 x 128 weight bytes, BN x 128 token bytes
// (128-byte swizzle) and both scale tiles. Warp 0 loads, warp 1 copies the scales to tensor memory
// and issues four MMAs, warps 2-5 read the sums back (a feature per lane). With a split each CTA
// owns some of the tile's tokens: every CTA writes its fp32 partial sums straight into the owners'
// shared memory, and after one cluster barrier the owners add them in rank order (a fixed
// order: same bits every time) and write y.
template <int BN>
struct Few {
  static constexpr int kA = 128 * 128, kB = BN * 128, kSf = 512;
  static constexpr int kStage = kA + kB + 2 * kSf;
  static constexpr int kMaxStages = 8;
  static constexpr int kSums = (BN + 8) * 512;          // partial sums of the tokens a CTA owns
  static constexpr int kThreads = 192;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr uint32_t kTmemCols = kAccCols + 8 * kMaxStages <= 128 ? 128 : 256;
  static constexpr int kBars = (2 * kMaxStages + 1) * 8 + 16;
  static constexpr int kFixed = kBars + 1024;           // barriers, and stages start on 1 KB
  static_assert(kStage % 1024 == 0, "swizzled stages start on 1 KB");
  static_assert(BN * 512 <= 3 * kStage, "unsplit sums take the place of the stages (at least 3)");
  static_assert(kAccCols + 8 * kMaxStages <= (int)kTmemCols, "tensor memory budget");
};

template <int BN>
__global__ void __launch_bounds__(Few<BN>::kThreads) fp8_few_kernel(const Fp8Args a, const int stages,
                                                                    const __grid_constant__ Fp8Maps M) {
  using C = Few<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint32_t splits, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(splits));
  rank = cluster_rank();
  // partial sums: behind the stages, or (no split: nobody else writes them) in their place
  float* sums = reinterpret_cast<float*>(smem + (splits > 1 ? stages * C::kStage : 0));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * C::kStage + (splits > 1 ? C::kSums : 0));
  uint64_t* empty = full + C::kMaxStages;
  uint64_t* done = empty + C::kMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int64_t tile = blockIdx.x / splits;
  const int64_t n0 = tile / a.n_tt * 128, m0 = tile % a.n_tt * BN;
  const int kb0 = (int)((int64_t)a.nkb * rank / splits), kb1 = (int)((int64_t)a.nkb * (rank + 1) / splits);
  const int ntok = (int)(a.m - m0 < BN ? a.m - m0 : BN);
  const int own = (int)((ntok + splits - 1) / splits);   // tokens a CTA of the cluster owns

  if (warp == 0 && elect_one_sync()) {
    // the first weights on their way to L2 while the previous kernel of the stream ends
    prefetch_tmap(&M.w); prefetch_tmap(&M.x);
    for (int kb = kb0; kb < kb1 && kb < kb0 + stages; ++kb) tma_2d_prefetch(&M.w, kb * 128, (int)n0);
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
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
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = fp8_wait(&empty[s], ph ^ 1, abort_flag, a.err, 20))) break;
        uint8_t* st = smem + (size_t)s * C::kStage;
        mbar_arrive_expect_tx(&full[s], C::kStage);
        tma_2d_g2s(st, &M.w, kb * 128, (int)n0, &full[s]);
        tma_2d_g2s(st + C::kA, &M.x, kb * 128, (int)m0, &full[s]);
        bulk_g2s(st + C::kA + C::kB, a.w_scales + (n0 / 128 * a.kgroups + kb / 4) * C::kSf, C::kSf, &full[s]);
        bulk_g2s(st + C::kA + C::kB + C::kSf, a.x_scales + (m0 / 128 * a.kgroups + kb / 4) * C::kSf, C::kSf,
                 &full[s]);
        ++issued;
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      if (!ok)                                           // copies in flight land before the CTA exits
        for (int j = issued > stages ? issued - stages : 0; j < issued; ++j)
          mbar_wait(&full[j % stages], (uint32_t)(j / stages) & 1, 1u << 20);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t kIdesc = idesc_mxf8(128, BN);
      const uint32_t sbase = smem_u32(smem);
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
          mma_mxf8<1>(tmem, da + 2 * k, db + 2 * k, id, sfa, sfb, acc);
          acc = 1;
        }
        if (kb + stages < kb1) mma_commit(&empty[s]);    // only where the producer waits for it
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      mma_commit(done);
      if (!ok) mbar_wait(done, 0, 1u << 22);             // MMAs in flight end before their memory goes
    }
    __syncwarp();
  }
  if (splits > 1) cluster_wait();                        // every CTA of the cluster runs
  if (warp >= 2 && __all_sync(0xffffffffu, fp8_wait(done, 0, abort_flag, a.err, 22))) {
    tc_fence_after();
    const int q4 = warp & 3, row = q4 * 32 + lane;       // tensor-memory lane = feature n0 + row
    const uint32_t taddr = tmem + ((uint32_t)(q4 * 32) << 16);
    const uint32_t mine = smem_u32(sums) + (rank * own * 128 + row) * 4;   // this rank's slot in an owner's sums
    int owner = 0, slot = 0;
    uint32_t dst = splits > 1 ? map_shared(mine, 0) : 0;
    constexpr int kCols = BN < 32 ? 16 : 32;
    for (int c0 = 0; c0 < ntok; c0 += kCols) {
      float v[kCols];
      if constexpr (kCols == 16) tmem_ld_32x32b_x16(taddr + c0, v);
      else tmem_ld_32x32b_x32(taddr + c0, v);
      tmem_wait_ld();
      if (splits > 1) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          if (c0 + j >= ntok) break;
          st_shared_cluster(dst + slot * 512, v[j]);
          if (++slot == own) { slot = 0; dst = map_shared(mine, min(++owner, (int)splits - 1)); }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kCols; ++j) sums[(c0 + j) * 128 + row] = v[j];   // c0 + j < BN
      }
    }
  }

  tc_fence_before();
  __syncwarp();
  if (splits > 1) cluster_sync();                        // every partial sum has landed
  else __syncthreads();
  // a warp per owned token, 4 features per lane
  const int f = lane * 4;
  const bool vec = n0 + 128 <= a.n && a.ldy % 4 == 0 && ((uintptr_t)a.y & 15) == 0;
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + f + i < a.n) bias[i] = load_as_float(a.bias, a.bias_dtype, n0 + f + i);
  const int t1 = min(own, ntok - (int)rank * own);
#pragma unroll 4
  for (int t = warp; t < t1; t += C::kThreads / 32) {
    float4 p = *reinterpret_cast<const float4*>(sums + t * 128 + f);
    for (uint32_t r = 1; r < splits; ++r) {
      const float4 q = *reinterpret_cast<const float4*>(sums + (r * own + t) * 128 + f);
      p.x += q.x; p.y += q.y; p.z += q.z; p.w += q.w;
    }
    const int64_t at = (m0 + (int)rank * own + t) * a.ldy + n0 + f;
    store4(a, at, n0 + f, p.x + bias[0], p.y + bias[1], p.z + bias[2], p.w + bias[3], vec);
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Shared memory a CTA may take so that one or two fit an SM (228 KB, 1 KB of it per CTA reserved).
constexpr int kSmemOne = 232448, kSmemTwo = 115712;

// Which split and pipeline a tile count gets: K is split over a cluster while that fills idle
// CTA slots and leaves every CTA at least 4 K blocks. Two CTAs per SM, but for 128-token tiles with a
// split, whose stages and partial sums take more than half an SM.
template <int BN>
int launch_few(const Fp8Args& a, const Fp8Maps& M, int dev, int nsm, cudaStream_t st) {
  using C = Few<BN>;
  static bool attr_set[64] = {false};
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(fp8_few_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOne));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t tiles = (a.n + 127) / 128 * a.n_tt;
  const int slots = BN == 128 ? nsm : 2 * nsm;
  int splits = (int)(slots / tiles < 8 ? slots / tiles : 8);
  if (splits > a.nkb / 4) splits = a.nkb / 4;
  if (splits < 1) splits = 1;
  const int sums = splits > 1 ? C::kSums : 0;
  const int room = (BN == 128 && tiles * splits <= nsm ? kSmemOne : kSmemTwo) - C::kFixed - sums;
  int stages = room / C::kStage < C::kMaxStages ? room / C::kStage : C::kMaxStages;
  const size_t smem = (size_t)stages * C::kStage + sums + C::kFixed;
  const int64_t grid = tiles * splits;
  FBFP_CHECK_ARG(grid < ((int64_t)1 << 31), "too many output tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FBFP_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_few_kernel<BN>, a, stages, M));
  FBFP_LAUNCH_CHECK("fp8_few_kernel");
  return FBFP_OK;
}

// ---------------------------------------------------------------------------------------
// Many tokens. Persistent CTA pairs (cta_group::2): a pair takes tiles of 256 tokens x BN features,
// tokens on the MMA's M side (128 per CTA), features on its N side (half of the weight rows in each
// CTA's shared memory), so that each SM loads 128 + BN / 2 rows of 128 bytes per K block for
// 128 x BN x 128 multiply-adds. Scale tiles are loaded once per 512 values of K, with the stage of
// the group's first K block, and copied to one of four slots of tensor memory in turn. A slot is
// written again 10 or more K blocks later where a tile has more than 8 (more than the stages in
// flight), else at least two tiles later (whose accumulator had to be drained first): either way
// the MMAs that read it have completed. A tile starts on a whole scale tile (features
// in steps of 128), which keeps the scales' tensor-memory addresses on multiples of 4 columns.
template <int BN>
struct Many {
  static constexpr int kHalfN = BN / 2;
  static constexpr int kChunks = BN / 128;                       // scale tiles of the features
  static constexpr int kA = 128 * 128, kB = kHalfN * 128, kSf = 512 * (1 + kChunks);
  static constexpr int kStage = kA + kB + (kSf + 1023) / 1024 * 1024;
  static constexpr int kStages = BN == 256 ? 6 : 8;
  static constexpr int kTurn = 32 * 17 * 4;                      // a warp's 32 x 16 words, rows 17 apart
  static constexpr int kBufs = BN == 256 ? 1 : 2;                // accumulators
  static constexpr int kSfCols = 4 * (1 + kChunks), kSfSlots = 4;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (4 + kEpiWarps);
  static constexpr uint32_t kTmemCols = 512, kSfCol0 = kBufs * BN;
  static constexpr int kData = kStages * kStage;
  static constexpr int kBarOff = kData + kEpiWarps * kTurn;
  static constexpr int kBars = 2 * kStages + 2 + 2 + 1;
  static constexpr size_t kSmem = kBarOff + kBars * 8 + 16 + 1024;
  static_assert(BN % 128 == 0 && kStage % 1024 == 0 && kTurn % 8 == 0, "features in whole scale tiles");
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

// One warp: 32 consecutive features, the first f0, of 32 consecutive tokens, one per lane (the
// first tok0; tokens from a.m on are not stored). vec: y's base and rows are 32-byte aligned, so
// each lane stores whole 32-byte sectors of its row; else the values turn through shared memory
// (`turn`) and the lanes store along the rows.
__device__ __forceinline__ void store_y32(const Fp8Args& a, int64_t tok0, int64_t f0, const float (&v)[32], bool vec,
                                          uint32_t* turn) {
  const int lane = threadIdx.x & 31;
  const int64_t row = tok0 + lane;
  uint32_t w[16];
  if (a.y_dtype != FBFP_F32) {
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
  }
  if (vec && f0 + 32 <= a.n) {
    if (row >= a.m) return;
    if (a.y_dtype == FBFP_F32) {
      float* p = reinterpret_cast<float*>(a.y) + row * a.ldy + f0;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p + 8 * h), "f"(v[8 * h]),
                     "f"(v[8 * h + 1]), "f"(v[8 * h + 2]), "f"(v[8 * h + 3]), "f"(v[8 * h + 4]), "f"(v[8 * h + 5]),
                     "f"(v[8 * h + 6]), "f"(v[8 * h + 7]) : "memory");
    } else {
      uint16_t* p = reinterpret_cast<uint16_t*>(a.y) + row * a.ldy + f0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p + 16 * h), "r"(w[8 * h]),
                     "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]), "r"(w[8 * h + 4]), "r"(w[8 * h + 5]),
                     "r"(w[8 * h + 6]), "r"(w[8 * h + 7]) : "memory");
    }
  } else if (a.y_dtype == FBFP_F32) {
    float* y = reinterpret_cast<float*>(a.y);
#pragma unroll
    for (int h = 0; h < 2; ++h) {                        // 16 columns at a time, two rows per store
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) turn[lane * 17 + i] = __float_as_uint(v[16 * h + i]);
      __syncwarp();
      const int64_t f = f0 + 16 * h + (lane & 15);
#pragma unroll 4
      for (int r = lane >> 4; r < 32; r += 2)
        if (tok0 + r < a.m && f < a.n) y[(tok0 + r) * a.ldy + f] = __uint_as_float(turn[r * 17 + (lane & 15)]);
    }
  } else {
    uint16_t* y = reinterpret_cast<uint16_t*>(a.y);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) turn[lane * 17 + i] = w[i];
    __syncwarp();
#pragma unroll 4
    for (int r = 0; r < 32; ++r)
      if (tok0 + r < a.m && f0 + lane < a.n)
        y[(tok0 + r) * a.ldy + f0 + lane] = reinterpret_cast<const uint16_t*>(turn + r * 17)[lane];
  }
}

template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Many<BN>::kThreads, 1)
fp8_many_kernel(const Fp8Args a, const __grid_constant__ Fp8Maps M) {
  using C = Many<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);   // used in CTA 0
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
    const int q4 = warp & 3, col0 = ((warp - 4) >> 2) * kCols;
    uint32_t* turn = reinterpret_cast<uint32_t*>(smem + C::kData + (warp - 4) * C::kTurn);
    const bool vec = ((uintptr_t)a.y & 31) == 0 && (a.ldy * (a.y_dtype == FBFP_F32 ? 4 : 2)) % 32 == 0;
    int buf = 0;
    uint32_t ph = 0;
    for (int64_t t = pair; t < tiles; t += pairs) {
      const int64_t tok0 = t % a.n_tt * 256 + 128 * rank + q4 * 32, n0 = t / a.n_tt * BN + col0;
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
        if (tok0 < a.m) store_y32(a, tok0, f0, v[c], vec, turn);
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
  a.x_scales = reinterpret_cast<const uint8_t*>(x_scales);
  a.w_scales = reinterpret_cast<const uint8_t*>(w_scales);
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
  const cudaStream_t st = as_stream(stream);
  if (many) {
    if ((rc = encode_2d(&M.xs, CU_TENSOR_MAP_DATA_TYPE_UINT32, x_scales, 128, (uint64_t)xt, 512, 128, 1,
                        CU_TENSOR_MAP_SWIZZLE_NONE)) != FBFP_OK) return rc;
    if ((rc = encode_2d(&M.ws, CU_TENSOR_MAP_DATA_TYPE_UINT32, w_scales, 128, (uint64_t)wt, 512, 128, 1,
                        CU_TENSOR_MAP_SWIZZLE_NONE)) != FBFP_OK) return rc;
    return launch_many<kManyN>(a, M, dev, nsm, st);
  }
  switch (bn) {
    case 16: return launch_few<16>(a, M, dev, nsm, st);
    case 32: return launch_few<32>(a, M, dev, nsm, st);
    case 64: return launch_few<64>(a, M, dev, nsm, st);
    default: return launch_few<128>(a, M, dev, nsm, st);
  }
}
