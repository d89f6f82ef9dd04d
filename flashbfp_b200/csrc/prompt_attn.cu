// prompt_attn.cu — causal attention of packed prompts on tcgen05: S = Q K^T into tensor memory, the
// softmax weights back into it as 16-bit operand, O += P V in tensor memory.
//
// A tile is 128 rows: `ntok` tokens of one sequence x the `hp` query heads that share a key/value head,
// so that grouped heads read keys and values once and a few tokens fill a tile. Keys and values are
// loaded in blocks of 128 keys (TMA). Heads of up to 128 values: a CTA takes two tiles over the same blocks;
// heads of up to 256: one, whose O fills half of tensor memory. Each tile has two score buffers, of 64 or 128
// keys, so that the next scores are made under this step's softmax. Roles: a warp loads; two warps issue MMAs,
// one per tile, or one the scores and one the products with the values (a wait costs an issuing warp some
// hundred cycles, and one warp's waits and issues in a row took longer than the MMAs themselves); four warps
// per tile hold one row a thread: scores from tensor memory, running maximum and sum, weights back. The grid
// has a CTA per tile (or two), longest first; a CTA that is done takes over the work of one that has not
// started, so that its next loads and first scores come under its last softmax and output.
//
// softmax: weights are 2^(s c - r), c = scaling log2(e), r the row's reference: its first step's
// maximum, raised (and O and the sum rescaled) only when a score comes out 2^8 above it, which leaves
// the quotient O / sum what it is (the lazily rescaled online softmax, published for attention on Blackwell). fp16
// weights carry a factor 2^6 that keeps small ones normal.
//
// Bound by the tensor cores and what feeds them from shared memory: at 256 values a block's two products read
// 192 KB and its loads write 128 KB (of 128 bytes a clock: 2500 clocks, the MMAs take 2048), at 128 the score
// MMAs of 64 keys read 6 KB in 32 clocks. Measured per block of 128 keys and SM (148 CTAs, a long axis): two
// tiles x 128 values 1.95 us (1270 TFLOP/s over all SMs), one tile x 256 values 1.63 us (1520). 8192 rows x 64
// heads of 128, fp16: 1.13-1.15 ms (953-970 TFLOP/s); 2048 rows x 16 heads of 256, bf16: 44.5 us; 128 rows over 32128
// keys: 86-88 us. Tried and left out: two teams of four warps for each tile (the softmax is not what is waited for),
// scores of 128 keys at once for heads of 128 (fewer bytes from shared memory, but no buffer to run ahead in).
#include <cuda.h>
#include <cmath>

#include "common.cuh"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {
using namespace sm100;

struct PromptArgs {
  int64_t rows, kv_rows, o_row, o_head, v_row, v_head, window;
  const int32_t *starts, *kv_starts;
  int wide;                    // out may be stored 32 bytes at a time
  int seqs, heads, hd, hp, ntok, head_blocks, group, splits;
  float c;                     // |scaling| log2(e)
  uint32_t negate;             // scaling < 0
  const void* v;
  void* out;
  float* part;                 // splits > 1: O / sum [split][hd / 8][head][row][8], then log2 of the sums [split][head][row]
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
  // Scores are made in steps of kKeys keys, two steps ahead of their softmax: each tile has two score buffers.
  static constexpr int kKeys = HDP <= 128 ? 64 : 128;
  static constexpr int kSub = kTile / kKeys;              // steps of a block
  static constexpr int kAhead = 2 / kSub;                 // blocks whose keys are loaded before the first values
  // A block's keys or values come in units. Up to 128 values a head: one unit. Up to 256: four units, of 64 of the
  // keys' values, or of 64 keys and 128 values, each given back as soon as it is used: the ring holds little
  // more than a block, and loads take as long as a block's products.
  static constexpr bool kFine = HDP == 256;
  static constexpr int kCols = HDP < 128 ? HDP : 128;     // values of a product's accumulator columns
  static constexpr int kUnit = kFine ? 16384 : kTile * HDP * 2;
  static constexpr int kPer = kFine ? 4 : 1;              // units per block
  static constexpr int kUnits = HDP == 64 ? 8 : kFine ? 10 : 5;           // depth of the ring
  static constexpr int kValueRows = kFine ? 64 : 128;     // keys of a unit of values
  static constexpr int kQ = kTile * HDP * 2;
  static constexpr int kSmem = kTiles * kQ + kUnits * kUnit + 1024;
  static constexpr int kSoft = 128 * kTiles;              // softmax threads
  static constexpr int kThreads = kSoft + 96;
  static constexpr uint32_t kO = 256;                     // first column of O; scores at 0 and 128
};

// What a CTA works on.
struct Work {
  int q0, len, k0, klen, tok0;  // the sequence's rows and keys, the first token
  int hb, split;                // block of heads, share of the keys
  int any;
};

struct Ctl {
  uint64_t q_full[2], q_empty, full[10], empty[10], s_full[2][2], p_full[2][2], v_here[2][2], o_done[2][2], voted[2], drain;
  uint64_t info_full[2], info_empty[2], next_full;
  uint4 next;                   // the answer to a request for another CTA's work
  Work info[2];                 // this tile's and the next one's, any = 0 behind the last
  uint32_t tmem;
  int abort, skip[2][2], vote[2][4];
};

// Out of line: the wait that does not end within some thousand polls.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, Ctl& ctl, int32_t* err, int site) {
  if (mbar_wait_second(bar, parity, &ctl.abort)) return true;
  *(volatile int*)&ctl.abort = 1;
  atomicExch(err, site);
  return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Ctl& ctl, int32_t* err, int site) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, 0;\n"
      "LOOP_%=:\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE_%=;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 q, n, 1024;\n\t"
      "@q bra LOOP_%=;\n"
      "DONE_%=:\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  if (__builtin_expect(ok != 0, 1)) return true;
  return wait_long(bar, parity, ctl, err, site);
}

__device__ __forceinline__ void tma_3d_g2s(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
      ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// The tensor core's instructions for a warp that goes the same way as a whole: one lane (`one`) issues, by a
// predicate and not a branch, so that descriptors are computed in uniform registers.
// D[tmem] (+)= A[smem] B[smem].
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc), "r"(one) : "memory");
}
// D[tmem] (+)= A[tmem] B[smem].
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(acc), "r"(one) : "memory");
}
__device__ __forceinline__ void commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
      ::"r"(smem_u32(bar)), "r"(one) : "memory");
}
// Values [keys][64] in 128-byte swizzled rows as the N-major operand: 8-key groups 1 KB apart, 64-value parts
// `part` bytes apart.
__device__ __forceinline__ uint64_t desc_values(uint32_t saddr, uint32_t part) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(part >> 4) << 16;
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

// 32 columns of this warp's 32 lanes; they may be used behind tmem_arrived.
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

// O += P V over keys l .. h of a step, for this thread's row: the weights come from tensor memory, the
// values from global memory. `fresh`: O holds nothing yet. (Out of line: only where a value is infinite or NaN.)
template <int HDP, typename T>
__device__ __noinline__ void add_seen(uint32_t o_at, uint32_t p_at, const T* v, int64_t v_row, int hd, int l, int h,
                                      bool fresh) {
#pragma unroll 1
  for (int d = 0; d < HDP; d += 32) {
    float o[32];
    tmem_load32(o_at + d, o);
    tmem_arrived<32>(o);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (fresh) o[i] = 0.f;
#pragma unroll 1
    for (int i = 0; i < Cfg<HDP>::kKeys / 2; ++i) {
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

// Where the search for a tile goes on: tiles of the sequences from b1 on come before, that many.
struct Cursor {
  int b1, before;
};
// CTA `index` of all tiles: the sequences' tiles from last to first, so that a prompt's longest tiles
// start first. By the loading warp. A CTA's indexes mostly ascend, and then all its searches together look at
// each sequence once. (Out of line: inlined, 8192 rows x 64 heads of 128 take 1.175 ms instead of 1.149, where one
// tile's call gains 0.2 us.)
__device__ __noinline__ Work find_work(const PromptArgs& a, int index, int toks, Cursor& cur) {
  const int lane = threadIdx.x & 31;
  Work w{0, 0, 0, 0, 0, 0, 0, 0};
  if (index < cur.before) cur = {a.seqs, 0};
#pragma unroll 1
  for (; cur.b1 > 0; cur.b1 -= 32) {
    const int b = cur.b1 - 1 - lane;
    int s0 = 0, s1 = 0, k0 = 0, k1 = 0;
    if (b >= 0) {
      s0 = __ldg(a.starts + b), s1 = __ldg(a.starts + b + 1), k0 = __ldg(a.kv_starts + b), k1 = __ldg(a.kv_starts + b + 1);
      s0 = min((int64_t)max(s0, 0), a.rows), s1 = min((int64_t)max(s1, s0), a.rows);
      k0 = min((int64_t)max(k0, 0), a.kv_rows), k1 = min((int64_t)max(k1, k0), a.kv_rows);
    }
    const int n = (s1 - s0 + toks - 1) / toks;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int place = index - cur.before - (sum - n);        // among the tiles of this lane's sequence
    const uint32_t who = __ballot_sync(0xffffffffu, place >= 0 && place < n);
    if (who) {
      const int src = __ffs(who) - 1;
      w.q0 = __shfl_sync(0xffffffffu, s0, src);
      w.len = __shfl_sync(0xffffffffu, s1, src) - w.q0;
      w.tok0 = __shfl_sync(0xffffffffu, n - 1 - place, src) * toks;
      w.k0 = __shfl_sync(0xffffffffu, k0, src);
      w.klen = __shfl_sync(0xffffffffu, k1, src) - w.k0;
      w.any = 1;
      return w;
    }
    cur.before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return w;
}

// Asks for the work of a CTA that has not been launched yet; the answer arrives on `bar`.
__device__ __forceinline__ void ask_next(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
// Whether there was such a CTA, and its block index.
__device__ __forceinline__ bool read_next(const uint4* answer, uint32_t& x, uint32_t& y) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%3];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, _, _}, r;\n\t}"
      : "=r"(ok), "=r"(x), "=r"(y) : "r"(smem_u32(answer)) : "memory");
  return ok != 0;
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
// The blocks of each tile of a CTA and of the CTA as a whole, lo .. hi - 1.
template <int TILES>
__device__ __forceinline__ void spans_of(const Work& w, const PromptArgs& a, Span (&span)[TILES], int& lo, int& hi) {
  lo = 1 << 30, hi = 0;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    span[t] = blocks_of(w, a, w.tok0 + t * a.ntok, a.ntok);
    if (span[t].hi > span[t].lo) lo = min(lo, span[t].lo), hi = max(hi, span[t].hi);
  }
  if (hi <= lo) lo = hi = 0;
  if (a.splits > 1) {
    const int n = hi - lo;
    const int from = lo + (int)((int64_t)n * w.split / a.splits), to = lo + (int)((int64_t)n * (w.split + 1) / a.splits);
    lo = from, hi = to;
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    span[t].lo = max(span[t].lo, lo), span[t].hi = min(span[t].hi, hi);
    if (span[t].hi <= span[t].lo) span[t] = {lo, lo};
  }
}
// 32 bytes at p, 32-byte aligned.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

template <int HDP, typename T>
__global__ void __launch_bounds__(Cfg<HDP>::kThreads, 1)
prompt_attn_kernel(const PromptArgs a, const __grid_constant__ PromptMaps M) {
  using C = Cfg<HDP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sq = smem_u32(smem), sring = sq + C::kTiles * C::kQ;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kLoad = C::kSoft / 32, kMma = kLoad + 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.q_full[i], 1);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&ctl.s_full[i][k], 1);
        mbar_init(&ctl.p_full[i][k], 4);
        mbar_init(&ctl.o_done[i][k], 1);
        mbar_init(&ctl.v_here[i][k], 1);
        ctl.skip[i][k] = 0;
      }
      mbar_init(&ctl.voted[i], 4);
      for (int k = 0; k < 4; ++k) ctl.vote[i][k] = 0;
      mbar_init(&ctl.info_full[i], 1);
      mbar_init(&ctl.info_empty[i], kLoad + 2);
    }
    for (int i = 0; i < 10; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], C::kTiles);           // (fine units are one warp's alone)
    }
    mbar_init(&ctl.q_empty, C::kTiles);
    mbar_init(&ctl.next_full, 1);
    mbar_init(&ctl.drain, 2);
    ctl.abort = 0;
    fence_mbar_init();
  }
  if (warp == kLoad && lane == 0) {
    prefetch_tmap(&M.q);
    prefetch_tmap(&M.k);
    prefetch_tmap(&M.v);
  }
  grid_dependency_wait();                            // before tensor memory is taken: the kernel before may hold some
  Cursor cur{a.seqs, 0};
  Work w0{0, 0, 0, 0, 0, 0, 0, 0};                   // the loading warp: this CTA's own tile
  if (warp == kMma) {                                // 512 columns, one CTA per SM
    tmem_alloc(&ctl.tmem, 512);
    tmem_relinquish();
  } else if (warp == kLoad) {
    w0 = find_work(a, blockIdx.x / a.head_blocks, a.ntok * C::kTiles, cur);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();                          // not before tensor memory is ours: a dependent may want some
  const uint32_t tmem = ctl.tmem;

  // The CTA goes on with the work of CTAs that have not started, tile after tile: the loads of the next tile and
  // its first scores come under the end of this one.
  const auto next_work = [&](int m, bool& ok) {      // tile m of this CTA, as the loading warp found it
    ok = __all_sync(0xffffffffu, wait(&ctl.info_full[m & 1], (uint32_t)(m >> 1) & 1, ctl, a.err, 43));
    Work w;                                          // (broadcast: the same in all lanes, for the compiler too)
    const int* from = reinterpret_cast<const int*>(&ctl.info[m & 1]);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Work) / 4); ++i)
      reinterpret_cast<int*>(&w)[i] = __shfl_sync(0xffffffffu, *(volatile const int*)(from + i), 0);
    if (lane == 0) mbar_arrive(&ctl.info_empty[m & 1]);
    return w;
  };

  int issued = 0, q_loads = 0, last = -1;            // loading: units and queries issued; this lane's last unit
  if (warp == kLoad) {
    const uint32_t q_bytes = (uint32_t)a.ntok * a.hp * 128 * (HDP / 64);
    uint32_t x = blockIdx.x, y = blockIdx.y;
    bool ok = true, more = true;
    int m = 0;                                       // tiles made known
    const auto tell = [&](const Work& w) {
      if (m >= 2) ok = __all_sync(0xffffffffu, wait(&ctl.info_empty[m & 1], (uint32_t)((m >> 1) - 1) & 1, ctl, a.err, 44));
      if (lane == 0 && ok) {
        ctl.info[m & 1] = w;
        mbar_arrive(&ctl.info_full[m & 1]);
      }
      ++m;
    };
#pragma unroll 1
    for (uint32_t asked = 0; more && ok; ++asked) {
      Work w = asked == 0 ? w0 : find_work(a, x / a.head_blocks, a.ntok * C::kTiles, cur);
      w.hb = x % a.head_blocks, w.split = y;
      if (w.any) {
        tell(w);
        const int kvh = w.hb / (a.group / a.hp), head0 = w.hb * a.hp;
        Span span[C::kTiles];
        int lo, hi;
        spans_of(w, a, span, lo, hi);
        if (hi > lo && ok) {
          // the units of block j, a lane each: one lane's waits and copies in a row would take as long as the
          // products that they feed
          const auto load = [&](const CUtensorMap* map, int j) {
            bool here = true;
            if (lane < C::kPer) {
              const int u = issued + lane, slot = u % C::kUnits;
              if (u >= C::kUnits) here = wait(&ctl.empty[slot], (uint32_t)(u / C::kUnits - 1) & 1, ctl, a.err, 32);
              if (here) {
                mbar_arrive_expect_tx(&ctl.full[slot], C::kUnit);
                const uint32_t to = sring + slot * C::kUnit, bar = smem_u32(&ctl.full[slot]);
                if constexpr (!C::kFine) {
                  for (int c = 0; c < HDP / 64; ++c) tma_3d_g2s(to + c * 16384, map, c * 64, kvh, w.k0 + j * kTile, bar);
                } else if (map == &M.k) {
                  tma_3d_g2s(to, map, lane * 64, kvh, w.k0 + j * kTile, bar);
                } else {
                  for (int c = 0; c < 2; ++c)
                    tma_3d_g2s(to + c * 8192, map, (lane & 1) * 128 + c * 64, kvh, w.k0 + j * kTile + (lane >> 1) * 64, bar);
                }
                last = u;
              }
            }
            ok = __all_sync(0xffffffffu, here);
            issued += C::kPer;
          };
          if (q_loads > 0) ok = __all_sync(0xffffffffu, wait(&ctl.q_empty, (uint32_t)(q_loads - 1) & 1, ctl, a.err, 45));
          if (ok) {
            if (lane == 0)
              for (int t = 0; t < C::kTiles; ++t) {
                mbar_arrive_expect_tx(&ctl.q_full[t], q_bytes);
                for (int c = 0; c < HDP / 64; ++c)
                  tma_3d_g2s(sq + t * C::kQ + c * 16384, &M.q, c * 64, head0, w.q0 + w.tok0 + t * a.ntok, smem_u32(&ctl.q_full[t]));
              }
            ++q_loads;
          }
          for (int j = lo; j < min(lo + C::kAhead, hi) && ok; ++j) load(&M.k, j);
          for (int j = lo; j < hi && ok; ++j) {
            load(&M.v, j);
            if (ok && j + C::kAhead < hi) load(&M.k, j + C::kAhead);
          }
        }
      }
      // asked for when this tile's loads are under way, no sooner: whoever is done first takes the next
      if (lane == 0) {
        mbar_arrive_expect_tx(&ctl.next_full, 16);
        ask_next(&ctl.next, &ctl.next_full);
      }
      if (!__all_sync(0xffffffffu, wait(&ctl.next_full, asked & 1, ctl, a.err, 46))) ok = false;
      if (ok) more = read_next(&ctl.next, x, y);
      fence_async_proxy();                           // read before the next answer lands
      __syncwarp();
    }
    if (ok) tell(Work{0, 0, 0, 0, 0, 0, 0, 0});
  } else if (warp >= kMma && C::kFine) {
    // Two warps issue, one the scores, one the products with the values: waits for units in between would keep
    // one from being ahead of the tensor cores. Each goes its way as a whole, one elected lane issues.
    const bool of_scores = warp == kMma;
    const uint32_t one = elect_one_sync();
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0), ring = __shfl_sync(0xffffffffu, sring, 0);
    const uint32_t id_s = idesc<T>(kTile, false) | (a.negate << 13), id_o = idesc<T>(C::kCols, true);
    const uint64_t q_desc = smem_desc_sw128(__shfl_sync(0xffffffffu, sq, 0), 1024);
    const uint64_t k_desc = smem_desc_sw128(ring, 1024), v_desc = desc_values(ring, C::kValueRows * 128);     // of slot 0
    uint32_t units = 0, g = 0;                       // units of the tiles before, steps so far
    int q_used = 0;
    bool ok = true;
#pragma unroll 1
    for (int m = 0; ok; ++m) {
      const Work w = next_work(m, ok);
      if (!ok || !w.any) break;
      Span span[C::kTiles];
      int lo, hi;
      spans_of(w, a, span, lo, hi);
      const uint32_t blocks = hi - lo;
      if (blocks == 0) continue;
      if (of_scores) {
        ok = __all_sync(0xffffffffu, wait(&ctl.q_full[0], q_used++ & 1, ctl, a.err, 34));
        for (uint32_t j = 0; j < blocks && ok; ++j, ++g) {
          // the product with the weights that the buffer held
          if (g >= 2) ok = __all_sync(0xffffffffu, wait(&ctl.o_done[0][g & 1], ((g >> 1) - 1) & 1, ctl, a.err, 33));
          uint32_t u = units + (j < 2 ? j : 2 * j - 1) * 4;
          uint32_t slot = u % C::kUnits, parity = (u / C::kUnits) & 1;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            if (ok) ok = __all_sync(0xffffffffu, wait(&ctl.full[slot], parity, ctl, a.err, 33));
            if (!ok) break;
            if (p == 0) tc_fence_after();
            const uint64_t qd = q_desc + (uint32_t)(p * 16384 / 16), kd = k_desc + slot * (C::kUnit / 16);
#pragma unroll
            for (int s = 0; s < 4; ++s) mma_ss(one, base + (g & 1) * C::kKeys, qd + s * 2, kd + s * 2, id_s, p + s > 0);
            commit(one, &ctl.empty[slot]);
            if (++slot == C::kUnits) slot = 0, parity ^= 1;
          }
          if (ok) commit(one, &ctl.s_full[0][g & 1]);
        }
        if (ok) commit(one, &ctl.q_empty);
      } else {
        for (uint32_t j = 0; j < blocks && ok; ++j, ++g) {
          uint32_t u = units + min(2 + 2 * j, blocks + j) * 4;
          uint32_t slot = u % C::kUnits, parity = (u / C::kUnits) & 1;
          bool skip = false;
          // A wait sees the parity of a phase and nothing else. The first units lie where the block's last keys
          // lay, units that this warp does not wait for: until those have landed, a wait for these would pass
          // on the phase before them. The block's scores are made: they have.
          ok = __all_sync(0xffffffffu, wait(&ctl.s_full[0][g & 1], (g >> 1) & 1, ctl, a.err, 47));
          if (!ok) break;
#pragma unroll
          for (int p = 0; p < 4; ++p) {              // keys 64 (p / 2) on, values 128 (p % 2) on
            if (ok) ok = __all_sync(0xffffffffu, wait(&ctl.full[slot], parity, ctl, a.err, 33));
            if (!ok) break;
            if (p == 0) {
              // the softmax may look at the values; all their units, where it does
              if (one) mbar_arrive(&ctl.v_here[0][g & 1]);
              ok = __all_sync(0xffffffffu, wait(&ctl.p_full[0][g & 1], (g >> 1) & 1, ctl, a.err, 35));
              if (!ok) break;
              tc_fence_after();
              skip = __any_sync(0xffffffffu, *(volatile int*)&ctl.skip[0][g & 1]);
            }
            const uint64_t vd = v_desc + slot * (C::kUnit / 16);
            if (!skip)
#pragma unroll
              for (int s = 0; s < 4; ++s)
                mma_ts(one, base + C::kO + (p & 1) * 128, base + (g & 1) * C::kKeys + ((p >> 1) * 4 + s) * 8, vd + s * 128, id_o,
                       j > 0 || p > 1 || s > 0);
            commit(one, &ctl.empty[slot]);
            if (++slot == C::kUnits) slot = 0, parity ^= 1;
          }
          if (ok) commit(one, &ctl.o_done[0][g & 1]);
        }
      }
      units += 2 * blocks * C::kPer;
    }
  } else if (warp >= kMma) {
    const int t = warp - kMma;                       // this warp's tile
    // The whole warp goes the same way, one elected lane issues: descriptors stay in uniform registers.
    const uint32_t one = elect_one_sync();
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0), ring = __shfl_sync(0xffffffffu, sring, 0);
    const uint32_t id_s = idesc<T>(C::kKeys, false) | (a.negate << 13), id_o = idesc<T>(C::kCols, true);
    const uint64_t q_desc = smem_desc_sw128(__shfl_sync(0xffffffffu, sq, 0), 1024);
    const uint64_t k_desc = smem_desc_sw128(ring, 1024), v_desc = desc_values(ring, C::kValueRows * 128);     // of slot 0
    // The ring: the next unit's slot, and the parity of its phase.
    uint32_t slot = 0, parity = 0;
    uint32_t made = 0, met = 0;                      // steps: scores made, values met (buffer: the lowest bit)
    int q_used = 0;
    bool ok = true;
    const auto arrived = [&]() {                     // the next block's units: the first's slot
      const uint32_t u = slot;
#pragma unroll
      for (int p = 0; p < C::kPer; ++p) {
        if (ok) ok = __all_sync(0xffffffffu, wait(&ctl.full[slot], parity, ctl, a.err, 33));
        if (++slot == C::kUnits) slot = 0, parity ^= 1;
      }
      return u;
    };
    const auto after = [&](uint32_t u, int p) { return u + p >= C::kUnits ? u + p - C::kUnits : u + p; };
    const auto release = [&](uint32_t u) {
#pragma unroll
      for (int p = 0; p < C::kPer; ++p) commit(one, &ctl.empty[after(u, p)]);
    };
    // A step's scores, later the product of its weights and values; `sub`: which keys of the block. Descriptors
    // count 16 bytes.
    const auto scores = [&](int sub, uint32_t u) {
      const uint32_t buf = made++ & 1;
      const uint32_t d = base + t * 128 + buf * C::kKeys;
#pragma unroll
      for (int p = 0; p < C::kPer; ++p) {
        const uint64_t qd = q_desc + (uint32_t)(t * C::kQ / 16);
        const uint64_t kd = k_desc + after(u, p) * (C::kUnit / 16) + (uint32_t)(sub * (C::kKeys * 128) / 16);
#pragma unroll
        for (int s = 0; s < C::kCols / 16; ++s) {
          const uint32_t at = ((s >> 2) * 16384 + (s & 3) * 32) / 16;
          mma_ss(one, d, qd + at, kd + at, id_s, p + s > 0);
        }
      }
      commit(one, &ctl.s_full[t][buf]);
    };
    const auto values = [&](int sub, uint32_t u, bool first) {
      const uint32_t buf = met & 1;
      ok = __all_sync(0xffffffffu, wait(&ctl.p_full[t][buf], (met++ >> 1) & 1, ctl, a.err, 35));
      if (!ok) return;
      tc_fence_after();
      const bool skip = __any_sync(0xffffffffu, *(volatile int*)&ctl.skip[t][buf]);
      if (!skip)
#pragma unroll
        for (int p = 0; p < C::kPer; ++p) {
          const uint64_t vd = v_desc + after(u, p) * (C::kUnit / 16) + (uint32_t)(sub * (C::kKeys * 128) / 16);
#pragma unroll
          for (int s = 0; s < C::kKeys / 16; ++s)
            mma_ts(one, base + C::kO + t * HDP + p * C::kCols, base + t * 128 + buf * C::kKeys + s * 8, vd + s * 128, id_o,
                   !first || s > 0);
        }
      commit(one, &ctl.o_done[t][buf]);
    };
#pragma unroll 1
    for (int m = 0; ok; ++m) {
      const Work w = next_work(m, ok);
      if (!ok || !w.any) break;
      Span span[C::kTiles];
      int lo, hi;
      spans_of(w, a, span, lo, hi);
      const int steps = (hi - lo) * C::kSub;
      if (steps == 0) continue;
      const Span mine = t == 0 ? span[0] : span[C::kTiles - 1];
      const int from = (mine.lo - lo) * C::kSub, to = (mine.hi - lo) * C::kSub;      // this tile's steps
      uint32_t uk = 0, uv = 0;
      if (ok) ok = __all_sync(0xffffffffu, wait(&ctl.q_full[t], q_used & 1, ctl, a.err, 34));
      ++q_used;
      for (int i = 0; i < min(2, steps) && ok; ++i) {
        if (i % C::kSub == 0) uk = arrived();
        if (ok && i >= from && i < to) scores(i % C::kSub, uk);
        if (ok && i % C::kSub == C::kSub - 1) release(uk);
      }
      if (steps <= 2 && ok) commit(one, &ctl.q_empty);
      for (int i = 0; i < steps && ok; ++i) {
        const bool in = i >= from && i < to;
        if (i % C::kSub == 0) {
          uv = arrived();
          if (!ok) break;
          if (one && in) mbar_arrive(&ctl.v_here[t][met / C::kSub & 1]);
        }
        if (in) values(i % C::kSub, uv, i == from);
        if (!ok) break;
        if (i % C::kSub == C::kSub - 1) release(uv);
        if (i + 2 < steps && (i + 2) % C::kSub == 0) uk = arrived();     // (keys are waited for no sooner than used)
        if (!ok) break;
        if (i + 2 >= from && i + 2 < to) scores(i % C::kSub, uk);       // (two steps on: the same part)
        if (i + 2 < steps && (i + 2) % C::kSub == C::kSub - 1) release(uk);
        if (i + 3 == steps) commit(one, &ctl.q_empty);
      }
    }
  } else {
    const int t = C::kTiles == 2 ? warp >> 2 : 0;    // this warp's tile
    const int r = threadIdx.x & 127;                 // this thread's row
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t o_at = tmem + C::kO + t * HDP + lanes;
    const float shift = kType<T> ? 0.f : 6.f;        // fp16 weights are 2^6 times as large
    uint32_t votes = 0, g = 0;                       // votes and steps so far
    int units = 0;                                   // units of the tiles so far
    bool ok = true;
#pragma unroll 1
    for (int m = 0; ok; ++m) {
    const Work w = next_work(m, ok);
    if (!ok || !w.any) break;
    Span span[C::kTiles];
    int lo, hi;
    spans_of(w, a, span, lo, hi);
    const int kvh = w.hb / (a.group / a.hp), head0 = w.hb * a.hp;
    const int tok = w.tok0 + t * a.ntok + r / a.hp, head = head0 + r % a.hp;
    const bool mine = r < a.ntok * a.hp && tok < w.len;
    const int place = mine ? w.klen - w.len + tok : -1;
    const int low = a.window > 0 ? (int)max((int64_t)place - a.window + 1, (int64_t)0) : 0;
    // all rows of the tile see keys all_low .. all_high
    const int tile0 = w.tok0 + t * a.ntok, tile1 = min(tile0 + a.ntok, w.len) - 1;
    const int all_high = w.klen - w.len + tile0;
    const int all_low = a.window > 0 ? (int)((int64_t)(w.klen - w.len + tile1) - a.window + 1) : 0;
    float ref = -INFINITY, sum0 = 0.f, sum1 = 0.f;   // reference (times c), sum of weights
    const int j0 = t == 0 ? span[0].lo : span[C::kTiles - 1].lo;
    const int i0 = j0 * C::kSub, steps = (t == 0 ? span[0].hi : span[C::kTiles - 1].hi) * C::kSub - i0;
#pragma unroll 1
    for (int n = 0; n < steps; ++n, ++g) {
      const int buf = g & 1;
      ok = __all_sync(0xffffffffu, wait(&ctl.s_full[t][buf], (g >> 1) & 1, ctl, a.err, 36));
      if (!ok) break;
      tc_fence_after();
      float s[C::kKeys];
      const uint32_t s_at = tmem + t * 128 + buf * C::kKeys + lanes;
#pragma unroll
      for (int i = 0; i < C::kKeys / 32; ++i) tmem_load32(s_at + 32 * i, s + 32 * i);
      tmem_arrived<C::kKeys>(s);
      const int key0 = (i0 + n) * C::kKeys;
      const bool cut = key0 + C::kKeys - 1 > all_high || key0 < all_low;      // the same in the whole tile
      const int h = place - key0, l = low - key0;     // the row sees keys l .. h of the step
      bool skip = false;
      if (cut) {
#pragma unroll
        for (int c = 0; c < C::kKeys; c += 32) {     // a bit for each key that is seen
          const int up = h - c, down = l - c;
          const uint32_t seen = (up >= 31 ? ~0u : up < 0 ? 0u : (2u << up) - 1) & (down <= 0 ? ~0u : down > 31 ? 0u : ~0u << down);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen >> i & 1)) s[c + i] = -INFINITY;
        }
      }
      float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < C::kKeys; ++i) tops[i & 3] = fmaxf(tops[i & 3], s[i]);
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * a.c;
      // the step before: its product
      const auto done_before = [&](int site) {
        return __all_sync(0xffffffffu, wait(&ctl.o_done[t][buf ^ 1], ((g - 1) >> 1) & 1, ctl, a.err, site));
      };
      if (n == 0) {
        ref = top;
      } else {
        const bool raise = top > ref + 8.f;
        if (__any_sync(0xffffffffu, raise)) {
          // O and the sum to the new reference, once the MMAs before have added to O
          ok = done_before(37);
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
      for (int i = 0; i < C::kKeys / 16; ++i) {
        uint32_t p[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float x = s[16 * i + e], y = s[16 * i + e + 1];
          fma2(x, y, a.c, less);
          x = ex2(x);
          y = ex2(y);
          add2(sum0, sum1, x, y);
          p[e / 2] = pack2(x, y, (const T*)nullptr);
        }
        tmem_st_32x32b_x8(s_at + 8 * i, p);
      }
      tmem_wait_st();
      if (cut) {
        // A weight of 0 does not silence an infinity or NaN in a value that its row does not see. Such
        // values of keys past the sequence's end, which no row sees, become 0; for others this step's
        // product is made here, over what each row sees.
        const int block = (i0 + n) / C::kSub - lo, blocks = hi - lo;
        const int unit = units + min(C::kAhead + 2 * block, blocks + block) * C::kPer;   // as they are loaded
        // Not every block's values are looked at, and a wait sees no more of a phase than its parity: so two
        // barriers take turns. The values two blocks before were here when the scores of this step's keys were asked
        // for, and those of the block before when these were told of.
        const uint32_t b = g / C::kSub;
        ok = wait(&ctl.v_here[t][b & 1], (b >> 1) & 1, ctl, a.err, 39);
        for (int p = 0; p < C::kPer && ok; ++p)
          ok = wait(&ctl.full[(unit + p) % C::kUnits], (uint32_t)((unit + p) / C::kUnits) & 1, ctl, a.err, 40);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // the tile's threads share the keys: this one's 16-byte pieces of key k's values, in an order free of
        // bank conflicts
        constexpr int kMine = HDP / 8 * C::kKeys / 128, kTurn = kMine < 8 ? kMine : 8;
        const int k = r % C::kKeys, first = r / C::kKeys * kMine;
        const int key = (i0 + n) % C::kSub * C::kKeys + k;                        // of the block
        uint8_t* const rows = smem + C::kTiles * C::kQ + key % C::kValueRows * 128;
        const int unit_k = unit + key / C::kValueRows * 2;
        const auto piece = [&](int i) {
          const int x = first + (i & ~(kTurn - 1)) + ((i + k) & (kTurn - 1));     // of HDP / 8
          return reinterpret_cast<uint4*>(rows + (unit_k + (x >> 4)) % C::kUnits * C::kUnit +
                                          ((x >> 3) & 1) * (C::kValueRows * 128) + ((x & 7) << 4));
        };
        uint32_t most = 0;                           // the largest bits, in halves
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const uint4 x = *piece(i);
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                         __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu)));
        }
        const uint32_t inf = kType<T> ? 0x7F80u : 0x7C00u;
        const bool odd = (most & 0xFFFFu) >= inf || (most >> 16) >= inf;
        const bool found = any_of_tile(odd, t, votes, ctl, a.err, ok);
        if (!ok) break;
        // zeros in the place of values past the end may be the other tile's, not fenced by its threads for this
        // tile's product
        if (C::kTiles == 2 && !found && key0 + C::kKeys > w.klen) fence_async_proxy();
        if (found) {
          const bool past = key0 + k >= w.klen;
          if (odd && past)
            for (int i = 0; i < kMine; ++i) *piece(i) = make_uint4(0, 0, 0, 0);
          fence_async_proxy();
          skip = any_of_tile(odd && !past, t, votes, ctl, a.err, ok);
          if (!ok) break;
          if (skip) {
            if (n > 0) ok = done_before(41);
            if (!ok) break;
            tc_fence_after();
            add_seen<HDP, T>(o_at, s_at, (const T*)a.v + (w.k0 + (int64_t)key0) * a.v_row + kvh * a.v_head, a.v_row, a.hd, l, h,
                             n == 0);
          }
        }
      }
      tc_fence_before();
      if (r == 0) *(volatile int*)&ctl.skip[t][buf] = skip;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.p_full[t][buf]);
    }
    if (!ok) break;
    units += 2 * (hi - lo) * C::kPer;
    if (steps > 0) {                                 // the last step's product, and all before it
      ok = __all_sync(0xffffffffu, wait(&ctl.o_done[t][(g - 1) & 1], ((g - 1) >> 1) & 1, ctl, a.err, 38));
      if (!ok) break;
      tc_fence_after();
    }
    const float sum = sum0 + sum1;
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);        // NaN stays
    const int64_t row = w.q0 + tok;
    if (a.splits > 1 && mine)
      a.lse[((int64_t)w.split * a.heads + head) * a.rows + row] = sum > 0.f ? lg2(sum) + ref - shift : (sum == 0.f ? -INFINITY : sum);
#pragma unroll 1
    for (int d = 0; d < HDP; d += 64) {
      float o[64];
      if (steps > 0) {
        tmem_load32(o_at + d, o);
        tmem_load32(o_at + d + 32, o + 32);
        tmem_arrived<64>(o);
      } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) o[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 64; ++i) o[i] *= inv;
      if (mine) {
        if (a.splits > 1) {
          // the tile's rows follow each other: whole lines (4.4 -> 2.6 us for 128 x 256 values)
          const int64_t step = (int64_t)a.heads * a.rows * 8;
          float* p = a.part + ((int64_t)w.split * (a.hd / 8) + d / 8) * step + ((int64_t)head * a.rows + row) * 8;
#pragma unroll
          for (int i = 0; i < 64; i += 8, p += step)
            if (d + i < a.hd) {
              uint32_t x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = __float_as_uint(o[i + e]);
              store32(p, x);
            }
        } else {
          T* p = (T*)a.out + row * a.o_row + head * a.o_head + d;
#pragma unroll
          for (int i = 0; i < 64; i += 16) {
            uint32_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = pack2(o[i + 2 * e], o[i + 2 * e + 1], p);
            if (a.wide) {                            // (values come in sixteens then)
              if (d + i < a.hd) store32(p + i, x);
            } else {
              if (d + i < a.hd) *reinterpret_cast<uint4*>(p + i) = make_uint4(x[0], x[1], x[2], x[3]);
              if (d + i + 8 < a.hd) *reinterpret_cast<uint4*>(p + i + 8) = make_uint4(x[4], x[5], x[6], x[7]);
            }
          }
        }
      }
    }
    tc_fence_before();                               // O is read before the next tile's products overwrite it
    }
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();                                   // every role has ended
  if (*(volatile int*)&ctl.abort) {                  // a wait gave up: loads and MMAs in flight land first
    if (warp == kLoad) {
      // a slot is loaded again only when its last load has been used: each lane's last units remain
      for (int u = last; u >= 0 && u > last - C::kUnits; u -= C::kPer)
        mbar_settle(&ctl.full[u % C::kUnits], (uint32_t)(u / C::kUnits) & 1);
      if (q_loads > 0 && lane == 0)
        for (int t = 0; t < C::kTiles; ++t) mbar_settle(&ctl.q_full[t], (uint32_t)(q_loads - 1) & 1);
    }
    if (warp >= kMma && elect_one_sync()) {          // the lanes that issued
      mma_commit(&ctl.drain);
      mbar_settle(&ctl.drain, 0);
    }
    __syncthreads();
  }
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits: weights 2^(lse - max) over the parts of a (row, head). A thread has 8 values; a warp 4 rows of a
// head x 8 such pieces, so that it reads and writes whole lines.
template <typename T>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptArgs a) {
  pdl_prologue();
  const int pieces = a.hd / 8;
  const int64_t quads = (a.rows + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t hq = (i >> 2) / pieces, head = hq / quads, row = (hq - head * quads) * 4 + (i & 3);
  const int piece = (int)((i >> 2) - hq * pieces);
  if (head >= a.heads || row >= a.rows) return;
  int lo = 0, hi = a.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.starts + mid) <= row) lo = mid;
    else hi = mid;
  }
  const int from = __ldg(a.starts + lo), to = __ldg(a.starts + lo + 1);
  const int64_t step = (int64_t)a.heads * a.rows;
  const float* const lse = a.lse + head * a.rows + row;
  float m = -INFINITY;
  bool nan = false;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float l = lse[s * step];
    nan |= l != l;
    m = fmaxf(m, l);
  }
  float sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float* p = a.part + (piece * step + head * a.rows + row) * 8;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s, p += pieces * step * 8) {
    const float l = lse[s * step];
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    if (l == -INFINITY) continue;                    // (nothing of this split: 0 all the same where nothing was seen)
    const float f = nan ? NAN : ex2(l - m);
    sum += f;
    o[0] += f * x.x, o[1] += f * x.y, o[2] += f * x.z, o[3] += f * x.w;
    o[4] += f * y.x, o[5] += f * y.y, o[6] += f * y.z, o[7] += f * y.w;
  }
  if (row < from || row >= to) return;               // rows of no sequence have no parts
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* const out = (T*)a.out + row * a.o_row + head * a.o_head + piece * 8;
  *reinterpret_cast<uint4*>(out) = make_uint4(pack2(o[0] * inv, o[1] * inv, out), pack2(o[2] * inv, o[3] * inv, out),
                                              pack2(o[4] * inv, o[5] * inv, out), pack2(o[6] * inv, o[7] * inv, out));
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

constexpr int64_t kNoWindow = 1 << 30;               // no sequence is longer

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
    const int64_t threads = (a.rows + 3) / 4 * 4 * a.heads * (a.hd / 8);
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
  if (window > kNoWindow) window = kNoWindow;
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
  FBFP_CHECK_ARG(std::isfinite(scaling * 1.4426950408889634f), "scaling %g is not finite, or its base-2 form is not", (double)scaling);
  if (window > kNoWindow) window = kNoWindow;        // before any sum with it
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15)
    return set_error(FBFP_ERR_ALIGN, "q, k, v and out must be 16-byte aligned");
  const Plan p = plan_of(rows, kv_rows, seqs, heads, kv_heads, head_dim, window);
  FBFP_CHECK_ARG(p.ctas <= 0x7FFFFFFF, "too many rows");
  const int64_t need = fbfp_prompt_attention_workspace_bytes(rows, kv_rows, seqs, heads, kv_heads, head_dim, window);
  FBFP_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 31) == 0),
                 "the workspace must be %lld bytes, 32-byte aligned", (long long)need);
  const int group = (int)(heads / kv_heads);
  PromptArgs a{rows, kv_rows, o_row, o_head, v_row, v_head, window, starts, kv_starts ? kv_starts : starts,
               head_dim % 16 == 0 && ((uintptr_t)out & 31) == 0 && ((o_row | o_head) & 15) == 0, (int)seqs, (int)heads,
               (int)head_dim, p.hp, p.ntok, p.head_blocks, group, p.splits,
               fmaxf(fabsf(scaling) * 1.4426950408889634f, 1e-30f), scaling < 0.f ? 1u : 0u, v, out, (float*)workspace,
               (float*)workspace + p.splits * rows * heads * head_dim, err};
  const CUtensorMapDataType dt = dtype == FBFP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  PromptMaps m;
  int st = encode_rows(&m.q, dt, q, head_dim, heads, rows, q_head, q_row, p.hp, p.ntok);
  if (!st) st = encode_rows(&m.k, dt, k, head_dim, kv_heads, kv_rows, k_head, k_row, 1, kTile);
  if (!st) st = encode_rows(&m.v, dt, v, head_dim, kv_heads, kv_rows, v_head, v_row, 1, head_dim > 128 ? 64 : kTile);
  if (st) return st;
  cudaStream_t s = as_stream(stream);
  if (head_dim <= 64) return dtype == FBFP_BF16 ? launch<64, __nv_bfloat16>(a, m, p, s) : launch<64, __half>(a, m, p, s);
  if (head_dim <= 128) return dtype == FBFP_BF16 ? launch<128, __nv_bfloat16>(a, m, p, s) : launch<128, __half>(a, m, p, s);
  return dtype == FBFP_BF16 ? launch<256, __nv_bfloat16>(a, m, p, s) : launch<256, __half>(a, m, p, s);
}
