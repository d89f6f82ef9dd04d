// prompt_attn.cu — causal attention of packed prompts on tcgen05: S = Q K^T into tensor memory, the
// softmax weights back into it as 16-bit operand, O += P V in tensor memory.
//
// A tile is 128 rows: `ntok` tokens of one sequence x the `hp` query heads that share a key/value head,
// so that grouped heads read keys and values once and a few tokens fill a tile. Its keys are taken in
// blocks of 128. Roles: a warp loads (TMA), a thread issues the MMAs, four warps per tile hold one row
// a thread: scores from tensor memory, running maximum and sum, weights back. Heads of up to 128
// values: a CTA takes two tiles, one's softmax runs under the other's MMAs. Heads of up to 256: one
// tile (its O fills half of tensor memory) with two score buffers, the next block's scores being made
// under this block's softmax.
//
// softmax: weights are 2^(s c - r), c = scaling log2(e), r the row's reference: its first block's
// maximum, raised (and O and the sum rescaled) only when a score comes out 2^8 above it, which leaves
// the quotient O / sum what it is. fp16 weights carry a factor 2^6 that keeps small ones normal.
#include <cuda.h>

#include "common.cuh"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {
using namespace sm100;

struct PromptArgs {
  int64_t rows, kv_rows, o_row, o_head, v_row, v_head, window;
  const int32_t *starts, *kv_starts;
  int seqs, heads, hd, hp, ntok, head_blocks, group, splits;
  float c;                     // |scaling| log2(e)
  uint32_t negate;             // scaling < 0
  const void* v;
  void* out;
  float* part;                 // splits > 1: O / sum [split][row][head][hd], then log2 of the sums [split][row][head]
  float* lse;
  int32_t* err;
};

struct PromptMaps {
  CUtensorMap q, k, v;
};

constexpr int kTile = 128;     // keys of a block, rows of a tile

template <int HDP>
struct Cfg {
  static constexpr int kTiles = HDP <= 128 ? 2 : 1;
  static constexpr int kAhead = HDP <= 128 ? 1 : 2;       // blocks whose scores are made ahead
  static constexpr int kCols = HDP < 128 ? HDP : 128;     // values of a unit
  static constexpr int kUnit = kTile * kCols * 2;        // a block's keys or values come in units
  static constexpr int kPer = HDP / kCols;                // units per block
  static constexpr int kUnits = HDP == 64 ? 8 : 5;        // depth of the ring
  static constexpr int kQ = kTile * HDP * 2;
  static constexpr int kSmem = kTiles * kQ + kUnits * kUnit + 1024;
  static constexpr int kSoft = 128 * kTiles;              // softmax threads
  static constexpr int kThreads = kSoft + 64;
  static constexpr uint32_t kO = 256;                     // first column of O; scores at 0 and 128
};

struct Ctl {
  uint64_t q_full[2], full[8], empty[8], s_full[2], p_full[2], v_here[2], o_done[2], voted[2], drain;
  uint32_t tmem;
  int abort, skip[2], vote[2][4];
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Ctl& ctl, int32_t* err, int site) {
  for (uint32_t it = 0; it < (1u << 16); ++it) {
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if ((it & 15) == 15 && *(volatile int*)&ctl.abort) return false;
  }
  *(volatile int*)&ctl.abort = 1;
  atomicExch(err, site);
  return false;
}
// After a wait gave up: what is in flight lands first (a bound of its own again, some 0.3 s).
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity) {
  for (uint32_t it = 0; it < (1u << 14); ++it)
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return;
}

__device__ __forceinline__ void tma_3d_g2s(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
      ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// D[tmem] (+)= A[smem] B[smem].
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc) : "memory");
}
// Values [128 keys][64] in 128-byte swizzled rows as the N-major operand: 8-key groups 1 KB apart,
// 64-value parts 16 KB apart.
__device__ __forceinline__ uint64_t desc_values(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(16384 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
template <typename T>
constexpr uint32_t kType = 0;                             // fp16
template <>
constexpr uint32_t kType<__nv_bfloat16> = 1;
template <typename T>
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_n_major) {
  return (1u << 4) | (kType<T> << 7) | (kType<T> << 10) | ((b_n_major ? 1u : 0u) << 16) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void fma2(float& a, float& b, float m, float add) {
  asm("{\n\t.reg .b64 x, m, c;\n\t"
      "mov.b64 x, {%0, %1};\n\tmov.b64 m, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
      "fma.rn.f32x2 x, x, m, c;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b) : "f"(m), "f"(add));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __float22bfloat162_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __float22half2_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// 32 columns of this warp's 32 lanes, usable at once.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr) : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// Loads have arrived: what uses the registers stays behind this.
template <int N>
__device__ __forceinline__ void tmem_arrived(float* v) {
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const float* v) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  tmem_st_32x32b_x32(addr, r);
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// Whether `x` holds for any of a tile's 128 rows: vote number `k` of tile t, whose rows all take part, with
// a bounded wait. A slot is cleared two votes before it is used again.
__device__ __forceinline__ bool any_of_tile(bool x, int t, uint32_t& k, Ctl& ctl, int32_t* err, bool& ok) {
  const bool any = __any_sync(0xffffffffu, x);
  if ((threadIdx.x & 31) == 0) {
    if (any) atomicOr(&ctl.vote[t][k & 3], 1);
    mbar_arrive(&ctl.voted[t]);
  }
  ok = __all_sync(0xffffffffu, wait(&ctl.voted[t], k & 1, ctl, err, 42));
  const bool r = *(volatile int*)&ctl.vote[t][k & 3] != 0;
  if ((threadIdx.x & 127) == 0) *(volatile int*)&ctl.vote[t][(k + 3) & 3] = 0;
  ++k;
  return r;
}

// O += P V over keys l .. h of a block, for this thread's row: the weights come from tensor memory, the
// values from global memory. (Out of line: only where a value is infinite or NaN.)
template <int HDP, typename T>
__device__ __noinline__ void add_seen(uint32_t o_at, uint32_t p_at, const T* v, int64_t v_row, int hd, int l, int h) {
#pragma unroll 1
  for (int d = 0; d < HDP; d += 32) {
    float o[32];
    tmem_load32(o_at + d, o);
    tmem_arrived<32>(o);
#pragma unroll 1
    for (int i = 0; i < kTile / 2; ++i) {
      uint32_t w;
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n" : "=r"(w) : "r"(p_at + i) : "memory");
      tmem_wait_ld();
      asm volatile("" : "+r"(w));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = 2 * i + e;
        if (key < l || key > h) continue;
        const uint16_t bits = (uint16_t)(w >> (16 * e));
        const float p = to_float(*reinterpret_cast<const T*>(&bits));
#pragma unroll
        for (int x = 0; x < 32; ++x)
          if (d + x < hd) o[x] = fmaf(p, to_float(v[key * v_row + d + x]), o[x]);
      }
      __syncwarp();
    }
    tmem_store32(o_at + d, o);
  }
  tmem_wait_st();
}

// What a CTA works on.
struct Work {
  int q0, len, k0, klen, tok0;  // the sequence's rows and keys, the first token
  bool any;
};

// CTA `index` of all tiles: the sequences' tiles from last to first, so that a prompt's longest tiles
// start first. Every warp finds it by itself.
__device__ __forceinline__ Work find_work(const PromptArgs& a, int index, int toks) {
  const int lane = threadIdx.x & 31;
  int total = 0;
  Work w{0, 0, 0, 0, 0, false};
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.seqs; b0 += 32) {
      const int b = b0 + lane;
      int s0 = 0, s1 = 0;
      if (b < a.seqs) {
        s0 = min((int64_t)max(__ldg(a.starts + b), 0), a.rows);
        s1 = min((int64_t)max(__ldg(a.starts + b + 1), s0), a.rows);
      }
      const int n = (s1 - s0 + toks - 1) / toks;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (pass == 1) {
        const int want = total - 1 - index;
        const bool mine = want >= before + sum - n && want < before + sum;
        const uint32_t who = __ballot_sync(0xffffffffu, mine);
        if (who) {
          const int src = __ffs(who) - 1;
          w.q0 = __shfl_sync(0xffffffffu, s0, src);
          w.len = __shfl_sync(0xffffffffu, s1, src) - w.q0;
          w.tok0 = (want - __shfl_sync(0xffffffffu, before + sum - n, src)) * toks;
          const int bb = b0 + src;
          w.k0 = min((int64_t)max(__ldg(a.kv_starts + bb), 0), a.kv_rows);
          w.klen = (int)min((int64_t)max(__ldg(a.kv_starts + bb + 1), w.k0), a.kv_rows) - w.k0;
          w.any = true;
          return w;
        }
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    total = before;
    if (index >= total) return w;
  }
  return w;
}

// Blocks of keys that tokens tok .. tok + n - 1 (those below len) see, cut to this split's share.
struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span blocks_of(const Work& w, const PromptArgs& a, int tok, int n) {
  const int last = min(tok + n, w.len) - 1;
  if (tok > last) return {0, 0};
  const int hi = w.klen - w.len + last + 1;                           // keys below this are seen
  if (hi <= 0) return {0, 0};
  const int first = w.klen - w.len + tok;
  const int lo = a.window > 0 ? (int)max((int64_t)first - a.window + 1, (int64_t)0) : 0;
  return {lo / kTile, (hi + kTile - 1) / kTile};
}

template <int HDP, typename T>
__global__ void __launch_bounds__(Cfg<HDP>::kThreads, 1)
prompt_attn_kernel(const PromptArgs a, const __grid_constant__ PromptMaps M) {
  using C = Cfg<HDP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sq = smem_u32(smem), sring = sq + C::kTiles * C::kQ;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  const int hb = blockIdx.x % a.head_blocks;
  const Work w = find_work(a, blockIdx.x / a.head_blocks, a.ntok * C::kTiles);
  if (!w.any) {
    grid_launch_dependents();
    return;
  }
  const int kvh = hb / (a.group / a.hp), head0 = hb * a.hp;
  // the blocks of each tile, and of the CTA
  Span span[C::kTiles];
  int lo = 1 << 30, hi = 0;
#pragma unroll
  for (int t = 0; t < C::kTiles; ++t) {
    span[t] = blocks_of(w, a, w.tok0 + t * a.ntok, a.ntok);
    if (span[t].hi > span[t].lo) lo = min(lo, span[t].lo), hi = max(hi, span[t].hi);
  }
  if (hi <= lo) lo = hi = 0;
  if (a.splits > 1) {
    const int n = hi - lo, s = blockIdx.y;
    const int from = lo + (int)((int64_t)n * s / a.splits), to = lo + (int)((int64_t)n * (s + 1) / a.splits);
    lo = from, hi = to;
  }
#pragma unroll
  for (int t = 0; t < C::kTiles; ++t) {
    span[t].lo = max(span[t].lo, lo), span[t].hi = min(span[t].hi, hi);
    if (span[t].hi <= span[t].lo) span[t] = {0, 0};
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.q_full[i], 1);
      mbar_init(&ctl.s_full[i], 1);
      mbar_init(&ctl.p_full[i], 4);
      mbar_init(&ctl.v_here[i], 1);
      mbar_init(&ctl.voted[i], 4);
      for (int k = 0; k < 4; ++k) ctl.vote[i][k] = 0;
      mbar_init(&ctl.o_done[i], 1);
      ctl.skip[i] = 0;
    }
    for (int i = 0; i < 8; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], 1);
    }
    mbar_init(&ctl.drain, 1);
    ctl.abort = 0;
    fence_mbar_init();
  }
  if (warp == C::kSoft / 32) {                       // the loading warp: 512 columns, one CTA per SM
    tmem_alloc(&ctl.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();                          // not before tensor memory is ours: a dependent may want some
  const uint32_t tmem = ctl.tmem;

  int issued = 0;                                    // loading: units issued
  if (warp == C::kSoft / 32) {
    if (lane == 0 && hi > lo) {
      prefetch_tmap(&M.q);
      prefetch_tmap(&M.k);
      prefetch_tmap(&M.v);
      const uint32_t q_bytes = (uint32_t)a.ntok * a.hp * 128 * (HDP / 64);
      const auto load_q = [&](int t) {
        mbar_arrive_expect_tx(&ctl.q_full[t], q_bytes);
        for (int c = 0; c < HDP / 64; ++c)
          tma_3d_g2s(sq + t * C::kQ + c * 16384, &M.q, c * 64, head0, w.q0 + w.tok0 + t * a.ntok, smem_u32(&ctl.q_full[t]));
      };
      bool ok = true;
      const auto load = [&](const CUtensorMap* map, int j) {        // the units of block j
        for (int p = 0; p < C::kPer && ok; ++p) {
          const int slot = issued % C::kUnits;
          if (issued >= C::kUnits) ok = wait(&ctl.empty[slot], (uint32_t)(issued / C::kUnits - 1) & 1, ctl, a.err, 32);
          if (!ok) return;
          mbar_arrive_expect_tx(&ctl.full[slot], C::kUnit);
          for (int c = 0; c < C::kCols / 64; ++c)
            tma_3d_g2s(sring + slot * C::kUnit + c * 16384, map, p * C::kCols + c * 64, kvh, w.k0 + j * kTile,
                       smem_u32(&ctl.full[slot]));
          ++issued;
        }
      };
      load_q(0);
      load(&M.k, lo);
      if (C::kTiles == 2) load_q(1);
      for (int j = lo + 1; j < min(lo + C::kAhead, hi); ++j) load(&M.k, j);
      for (int j = lo; j < hi && ok; ++j) {
        load(&M.v, j);
        if (j + C::kAhead < hi) load(&M.k, j + C::kAhead);
      }
    }
  } else if (warp == C::kSoft / 32 + 1) {
    if (lane == 0 && hi > lo) {
      const uint32_t id_s = idesc<T>(kTile, false) | (a.negate << 13), id_o = idesc<T>(C::kCols, true);
      int used = 0;                                  // units taken, in the order of their loading
      bool ok = true;
      const auto arrived = [&]() {                   // the next block's units: the first's number
        const int u = used;
        for (int p = 0; p < C::kPer && ok; ++p, ++used)
          ok = wait(&ctl.full[used % C::kUnits], (uint32_t)(used / C::kUnits) & 1, ctl, a.err, 33);
        return u;
      };
      const auto release = [&](int u) {
        for (int p = 0; p < C::kPer; ++p) mma_commit(&ctl.empty[(u + p) % C::kUnits]);
      };
      const auto scores = [&](int t, int buf, int u) {
        for (int p = 0; p < C::kPer; ++p) {
          const uint32_t kb = sring + ((u + p) % C::kUnits) * C::kUnit;
          for (int s = 0; s < C::kCols / 16; ++s) {
            const uint32_t at = (s >> 2) * 16384 + (s & 3) * 32;
            mma_ss(tmem + buf * 128, smem_desc_sw128(sq + t * C::kQ + p * 32768 + at, 1024), smem_desc_sw128(kb + at, 1024),
                   id_s, p + s > 0);
          }
        }
        mma_commit(&ctl.s_full[buf]);
      };
      const auto values = [&](int t, int buf, int u, bool skip) {
        if (!skip)
          for (int p = 0; p < C::kPer; ++p) {
            const uint32_t vb = sring + ((u + p) % C::kUnits) * C::kUnit;
            for (int s = 0; s < kTile / 16; ++s)
              mma_ts(tmem + C::kO + t * HDP + p * C::kCols, tmem + buf * 128 + s * 8, desc_values(vb + s * 2048), id_o, 1);
          }
        mma_commit(&ctl.o_done[t]);
      };
      uint32_t p_seen[2] = {0, 0};
      if constexpr (C::kTiles == 2) {
        ok = wait(&ctl.q_full[0], 0, ctl, a.err, 34);
        const int u0 = ok ? arrived() : 0;
        if (ok && span[0].lo == lo && span[0].hi > lo) scores(0, 0, u0);
        if (ok) ok = wait(&ctl.q_full[1], 0, ctl, a.err, 34);
        if (ok && span[1].lo == lo && span[1].hi > lo) scores(1, 1, u0);
        if (ok) release(u0);
        for (int j = lo; j < hi && ok; ++j) {
          const int uv = arrived();
          if (!ok) break;
          for (int t = 0; t < 2; ++t)
            if (j >= span[t].lo && j < span[t].hi) mbar_arrive(&ctl.v_here[t]);
          const int uk = j + 1 < hi ? arrived() : 0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && j >= span[t].lo && j < span[t].hi) {
              ok = wait(&ctl.p_full[t], p_seen[t]++ & 1, ctl, a.err, 35);
              if (!ok) break;
              tc_fence_after();
              values(t, t, uv, *(volatile int*)&ctl.skip[t]);
            }
            if (t == 1 && ok) release(uv);
            if (ok && j + 1 >= span[t].lo && j + 1 < span[t].hi) scores(t, t, uk);
          }
          if (ok && j + 1 < hi) release(uk);
        }
      } else {
        ok = wait(&ctl.q_full[0], 0, ctl, a.err, 34);
        for (int j = lo; j < min(lo + 2, hi) && ok; ++j) {
          const int u = arrived();
          if (!ok) break;
          scores(0, (j - lo) & 1, u);
          release(u);
        }
        for (int j = lo; j < hi && ok; ++j) {
          const int buf = (j - lo) & 1;
          const int uv = arrived();
          if (!ok) break;
          mbar_arrive(&ctl.v_here[0]);
          ok = wait(&ctl.p_full[buf], p_seen[buf]++ & 1, ctl, a.err, 35);
          if (!ok) break;
          tc_fence_after();
          values(0, buf, uv, *(volatile int*)&ctl.skip[buf]);
          release(uv);
          if (j + 2 < hi) {
            const int u = arrived();
            if (!ok) break;
            scores(0, buf, u);
            release(u);
          }
        }
      }
    }
  } else {
    const int t = C::kTiles == 2 ? warp >> 2 : 0;    // this warp's tile
    const int r = threadIdx.x & 127;                 // this thread's row
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t o_at = tmem + C::kO + t * HDP + lanes;
    const int tok = w.tok0 + t * a.ntok + r / a.hp, head = head0 + r % a.hp;
    const bool mine = r < a.ntok * a.hp && tok < w.len;
    const int place = mine ? w.klen - w.len + tok : -1;
    const int low = a.window > 0 ? (int)max((int64_t)place - a.window + 1, (int64_t)0) : 0;
    // all rows of the tile see keys all_low .. all_high
    const int tile0 = w.tok0 + t * a.ntok, tile1 = min(tile0 + a.ntok, w.len) - 1;
    const int all_high = w.klen - w.len + tile0;
    const int all_low = a.window > 0 ? (int)((int64_t)(w.klen - w.len + tile1) - a.window + 1) : 0;
    const float shift = kType<T> ? 0.f : 6.f;        // fp16 weights are 2^6 times as large
    float ref = -INFINITY, sum0 = 0.f, sum1 = 0.f;   // reference (times c), sum of weights
    uint32_t votes = 0;
    bool ok = true;
    const int j0 = t == 0 ? span[0].lo : span[C::kTiles - 1].lo, j1 = t == 0 ? span[0].hi : span[C::kTiles - 1].hi;
    if (j1 > j0) {
      float z[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) z[i] = 0.f;
#pragma unroll 1
      for (int d = 0; d < HDP; d += 32) tmem_store32(o_at + d, z);
    }
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      const int n = j - j0;                          // blocks before
      const int buf = C::kTiles == 2 ? t : n & 1;
      const uint32_t phase = C::kTiles == 2 ? n & 1 : (n >> 1) & 1;
      ok = __all_sync(0xffffffffu, wait(&ctl.s_full[buf], phase, ctl, a.err, 36));
      if (!ok) break;
      tc_fence_after();
      float s[128];
      const uint32_t s_at = tmem + buf * 128 + lanes;
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_load32(s_at + 32 * i, s + 32 * i);
      tmem_arrived<128>(s);
      const int key0 = j * kTile;
      const bool cut = key0 + kTile - 1 > all_high || key0 < all_low;        // the same in the whole tile
      const int h = place - key0, l = low - key0;     // the row sees keys l .. h of the block
      bool skip = false;
      if (cut) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > h || i < l) s[i] = -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 128; ++i) top = fmaxf(top, s[i]);
      top *= a.c;
      if (n == 0) {
        ref = top;
      } else {
        const bool raise = top > ref + 8.f;
        if (__any_sync(0xffffffffu, raise)) {
          // O and the sum to the new reference, once the MMAs before have added to O
          ok = __all_sync(0xffffffffu, wait(&ctl.o_done[t], (uint32_t)(n - 1) & 1, ctl, a.err, 37));
          if (!ok) break;
          tc_fence_after();
          const float f = raise ? ex2(ref - top) : 1.f;              // 0 where there was none
          if (raise) ref = top;
          sum0 *= f;
          sum1 *= f;
#pragma unroll 1
          for (int d = 0; d < HDP; d += 32) {
            float o[32];
            tmem_load32(o_at + d, o);
            tmem_arrived<32>(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= f;
            tmem_store32(o_at + d, o);
          }
        }
      }
      const float less = ref == -INFINITY ? 0.f : shift - ref;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float x = s[32 * i + e], y = s[32 * i + e + 1];
          fma2(x, y, a.c, less);
          x = ex2(x);
          y = ex2(y);
          add2(sum0, sum1, x, y);
          p[e / 2] = pack2(x, y, (const T*)nullptr);
        }
        uint32_t p0[8], p1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p0[e] = p[e], p1[e] = p[8 + e];
        tmem_st_32x32b_x8(s_at + 16 * i, p0);
        tmem_st_32x32b_x8(s_at + 16 * i + 8, p1);
      }
      tmem_wait_st();
      if (cut) {
        // A weight of 0 does not silence an infinity or NaN in a value that its row does not see. Such
        // values of keys past the sequence's end, which no row sees, become 0; for others this block's
        // product is made here, over what each row sees.
        const int block = j - lo, blocks = hi - lo;
        const int unit = min(C::kAhead + 2 * block, blocks + block) * C::kPer;   // as they are loaded
        ok = wait(&ctl.v_here[t], n & 1, ctl, a.err, 39);
        for (int p = 0; p < C::kPer && ok; ++p)
          ok = wait(&ctl.full[(unit + p) % C::kUnits], (uint32_t)((unit + p) / C::kUnits) & 1, ctl, a.err, 40);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint32_t most = 0;                           // of the bits of key r's values, in halves
#pragma unroll
        for (int i = 0; i < HDP / 8; ++i) {
          const int part = i >> 3;                   // 64 values; their 16-byte pieces in an order free of conflicts
          const uint4 x = *reinterpret_cast<const uint4*>(smem + C::kTiles * C::kQ + (unit + part / 2) % C::kUnits * C::kUnit +
                                                          (part & 1) * 16384 + r * 128 + (((i + r) & 7) << 4));
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                         __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu)));
        }
        const uint32_t inf = kType<T> ? 0x7F80u : 0x7C00u;
        const bool odd = (most & 0xFFFFu) >= inf || (most >> 16) >= inf;
        const bool found = any_of_tile(odd, t, votes, ctl, a.err, ok);
        if (!ok) break;
        if (found) {
          const bool past = key0 + r >= w.klen;
          if (odd && past)
            for (int i = 0; i < HDP / 8; ++i)
              *reinterpret_cast<uint4*>(smem + C::kTiles * C::kQ + (unit + (i >> 4)) % C::kUnits * C::kUnit +
                                        ((i >> 3) & 1) * 16384 + r * 128 + ((i & 7) << 4)) = make_uint4(0, 0, 0, 0);
          fence_async_proxy();
          skip = any_of_tile(odd && !past, t, votes, ctl, a.err, ok);
          if (!ok) break;
          if (skip) {
            if (n > 0) ok = __all_sync(0xffffffffu, wait(&ctl.o_done[t], (uint32_t)(n - 1) & 1, ctl, a.err, 41));
            if (!ok) break;
            tc_fence_after();
            add_seen<HDP, T>(o_at, s_at, (const T*)a.v + (w.k0 + (int64_t)key0) * a.v_row + kvh * a.v_head, a.v_row, a.hd, l, h);
          }
        }
      }
      tc_fence_before();
      if (r == 0) *(volatile int*)&ctl.skip[buf] = skip;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.p_full[buf]);
    }
    // the last block's product; with two score buffers the one before it may be on its way too
    for (int n = max(j1 - j0 - C::kAhead, 0); n < j1 - j0 && ok; ++n)
      ok = __all_sync(0xffffffffu, wait(&ctl.o_done[t], (uint32_t)n & 1, ctl, a.err, 38));
    if (ok) {
      tc_fence_after();
      const float sum = sum0 + sum1;
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);      // NaN stays
      const int64_t row = w.q0 + tok;
      if (a.splits > 1 && mine)
        a.lse[((int64_t)blockIdx.y * a.rows + row) * a.heads + head] = sum > 0.f ? lg2(sum) + ref - shift : (sum == 0.f ? -INFINITY : sum);
#pragma unroll 1
      for (int d = 0; d < HDP; d += 32) {
        float o[32];
        if (j1 > j0) {
          tmem_load32(o_at + d, o);
          tmem_arrived<32>(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] *= inv;
        if (mine) {
          if (a.splits > 1) {
            float* p = a.part + (((int64_t)blockIdx.y * a.rows + row) * a.heads + head) * a.hd + d;
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (d + i < a.hd) *reinterpret_cast<float4*>(p + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          } else {
            T* p = (T*)a.out + row * a.o_row + head * a.o_head + d;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              if (d + i < a.hd)
                *reinterpret_cast<uint4*>(p + i) =
                    make_uint4(pack2(o[i], o[i + 1], p), pack2(o[i + 2], o[i + 3], p), pack2(o[i + 4], o[i + 5], p),
                               pack2(o[i + 6], o[i + 7], p));
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();                                   // every role has ended
  if (*(volatile int*)&ctl.abort) {                  // a wait gave up: loads and MMAs in flight land first
    if (warp == C::kSoft / 32 && lane == 0) {
      for (int u = issued > C::kUnits ? issued - C::kUnits : 0; u < issued; ++u)
        settle(&ctl.full[u % C::kUnits], (uint32_t)(u / C::kUnits) & 1);
      if (hi > lo)
        for (int t = 0; t < C::kTiles; ++t) settle(&ctl.q_full[t], 0);
    }
    if (warp == C::kSoft / 32 + 1 && lane == 0) {
      mma_commit(&ctl.drain);
      settle(&ctl.drain, 0);
    }
    __syncthreads();
  }
  if (warp == C::kSoft / 32) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits: weights 2^(lse - max) over the parts of a (row, head); a thread per 4 values.
template <typename T>
__global__ void prompt_join_kernel(const PromptArgs a) {
  pdl_prologue();
  const int per = a.hd / 4;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t rh = i / per;
  const int d = (int)(i - rh * per) * 4;
  if (rh >= a.rows * a.heads) return;
  const int64_t row = rh / a.heads;
  // rows of no sequence have no parts
  int lo = 0, hi = a.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.starts + mid) <= row) lo = mid;
    else hi = mid;
  }
  if (row < __ldg(a.starts + lo) || row >= __ldg(a.starts + lo + 1)) return;
  const int64_t step = a.rows * a.heads;
  float m = -INFINITY;
  bool nan = false;
  for (int s = 0; s < a.splits; ++s) {
    const float l = a.lse[s * step + rh];
    nan |= l != l;
    m = fmaxf(m, l);
  }
  float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float l = a.lse[s * step + rh];
    if (l == -INFINITY) continue;
    const float f = nan ? NAN : ex2(l - m);
    const float4 p = *reinterpret_cast<const float4*>(a.part + (s * step + rh) * a.hd + d);
    sum += f;
    o[0] += f * p.x, o[1] += f * p.y, o[2] += f * p.z, o[3] += f * p.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* p = (T*)a.out + row * a.o_row + (rh - row * a.heads) * a.o_head + d;
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(o[0] * inv, o[1] * inv, p), pack2(o[2] * inv, o[3] * inv, p));
}

// How a call is cut: heads of a tile (the largest divisor of a group that a tile holds), its tokens,
// and the splits of the keys where the tiles do not fill the SMs.
struct Plan {
  int hp, ntok, tiles, head_blocks, splits;
  int64_t ctas;
};
Plan plan_of(int64_t rows, int64_t kv_rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t hd, int64_t window) {
  Plan p;
  const int group = (int)(heads / kv_heads);
  p.hp = group < kTile ? group : kTile;
  while (group % p.hp) --p.hp;
  p.ntok = kTile / p.hp;
  p.tiles = hd <= 128 ? 2 : 1;
  p.head_blocks = (int)heads / p.hp;
  const int64_t toks = (int64_t)p.ntok * p.tiles;
  // each sequence that has rows ends in a tile of its own
  p.ctas = (rows + (seqs < rows ? seqs : rows) * (toks - 1)) / toks * p.head_blocks;
  int64_t reach = kv_rows;                                             // keys of a CTA at most
  if (window > 0 && window + toks < reach) reach = window + toks;
  const int64_t blocks = (reach + kTile - 1) / kTile;
  // fill 148 SMs, but leave each split four blocks: below that its own start outweighs its work
  int64_t s = 148 / p.ctas;
  if (s > blocks / 4) s = blocks / 4;
  p.splits = s < 1 ? 1 : (int)s;
  return p;
}

template <int HDP, typename T>
int launch(const PromptArgs& a, const PromptMaps& m, const Plan& p, cudaStream_t st) {
  auto kernel = prompt_attn_kernel<HDP, T>;
  static bool set[64];
  int dev = 0;
  FBFP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HDP>::kSmem));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  FBFP_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)p.ctas, (unsigned)p.splits), dim3(Cfg<HDP>::kThreads),
                           (size_t)Cfg<HDP>::kSmem, st, a, m));
  FBFP_LAUNCH_CHECK("prompt_attn_kernel");
  if (p.splits > 1) {
    const int64_t threads = a.rows * a.heads * (a.hd / 4);
    FBFP_CUDA_TRY(launch_pdl(prompt_join_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a));
    FBFP_LAUNCH_CHECK("prompt_join_kernel");
  }
  return FBFP_OK;
}

// Rows of heads as a tensor of (value, head, row).
int encode_rows(CUtensorMap* m, CUtensorMapDataType dt, const void* base, int64_t hd, int64_t heads, int64_t rows,
                int64_t head_stride, int64_t row_stride, int box_heads, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(FBFP_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = encode_tiled(fn, m, dt, 3u, const_cast<void*>(base), dims, strides, box, es,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FBFP_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return FBFP_OK;
}

}  // namespace
}  // namespace fbfp

using namespace fbfp;

extern "C" int64_t fbfp_prompt_attention_workspace_bytes(int64_t rows, int64_t kv_rows, int64_t seqs, int64_t heads,
                                                         int64_t kv_heads, int64_t head_dim, int64_t window) {
  if (rows < 1 || kv_rows < 1 || seqs < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1) return -1;
  const Plan p = plan_of(rows, kv_rows, seqs, heads, kv_heads, head_dim, window);
  return p.splits > 1 ? p.splits * rows * heads * (head_dim + 1) * 4 : 0;
}

extern "C" int fbfp_prompt_attention(const void* q, const void* k, const void* v, int dtype, int64_t rows,
                                     int64_t kv_rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                     int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row,
                                     int64_t v_head, const int32_t* starts, const int32_t* kv_starts, int64_t window,
                                     float scaling, void* out, int64_t o_row, int64_t o_head, void* workspace,
                                     int64_t workspace_bytes, int32_t* err, void* stream) {
  FBFP_CHECK_ARG(q && k && v && starts && out && err, "null pointer");
  FBFP_CHECK_ARG(dtype == FBFP_BF16 || dtype == FBFP_F16, "bad dtype %d (bf16 or fp16)", dtype);
  FBFP_CHECK_ARG(rows >= 1 && rows < (1 << 30) && kv_rows >= 1 && kv_rows < (1 << 30) && seqs >= 1 && seqs <= 65535,
                 "bad sizes (%lld rows, %lld key rows, %lld sequences)", (long long)rows, (long long)kv_rows,
                 (long long)seqs);
  FBFP_CHECK_ARG(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 65535, "%lld heads over %lld",
                 (long long)heads, (long long)kv_heads);
  FBFP_CHECK_ARG(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, "head_dim %lld is not a multiple of 8 up to 256",
                 (long long)head_dim);
  FBFP_CHECK_ARG(q_row >= 0 && q_head >= 0 && k_row >= 0 && k_head >= 0 && v_row >= 0 && v_head >= 0 && o_row >= 0 &&
                     o_head >= 0 && ((q_row | q_head | k_row | k_head | v_row | v_head | o_row | o_head) & 7) == 0,
                 "strides must be multiples of 8");
  FBFP_CHECK_ARG(window >= 0, "negative window");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15)
    return set_error(FBFP_ERR_ALIGN, "q, k, v and out must be 16-byte aligned");
  const Plan p = plan_of(rows, kv_rows, seqs, heads, kv_heads, head_dim, window);
  FBFP_CHECK_ARG(p.ctas <= 0x7FFFFFFF, "too many rows");
  const int64_t need = fbfp_prompt_attention_workspace_bytes(rows, kv_rows, seqs, heads, kv_heads, head_dim, window);
  FBFP_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                 "the workspace must be %lld bytes, 16-byte aligned", (long long)need);
  const int group = (int)(heads / kv_heads);
  if (window > (1 << 30)) window = 1 << 30;          // no longer than any sequence
  PromptArgs a{rows, kv_rows, o_row, o_head, v_row, v_head, window, starts, kv_starts ? kv_starts : starts, (int)seqs, (int)heads,
               (int)head_dim, p.hp, p.ntok, p.head_blocks, group, p.splits,
               fmaxf(fabsf(scaling) * 1.4426950408889634f, 1e-30f), scaling < 0.f ? 1u : 0u, v, out, (float*)workspace,
               (float*)workspace + p.splits * rows * heads * head_dim, err};
  const CUtensorMapDataType dt = dtype == FBFP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  PromptMaps m;
  int st = encode_rows(&m.q, dt, q, head_dim, heads, rows, q_head, q_row, p.hp, p.ntok);
  if (!st) st = encode_rows(&m.k, dt, k, head_dim, kv_heads, kv_rows, k_head, k_row, 1, kTile);
  if (!st) st = encode_rows(&m.v, dt, v, head_dim, kv_heads, kv_rows, v_head, v_row, 1, kTile);
  if (st) return st;
  cudaStream_t s = as_stream(stream);
  if (head_dim <= 64) return dtype == FBFP_BF16 ? launch<64, __nv_bfloat16>(a, m, p, s) : launch<64, __half>(a, m, p, s);
  if (head_dim <= 128) return dtype == FBFP_BF16 ? launch<128, __nv_bfloat16>(a, m, p, s) : launch<128, __half>(a, m, p, s);
  return dtype == FBFP_BF16 ? launch<256, __nv_bfloat16>(a, m, p, s) : launch<256, __half>(a, m, p, s);
}
