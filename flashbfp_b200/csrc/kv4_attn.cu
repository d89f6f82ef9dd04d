// kv4_attn.cu — attention of the newest rows of each sequence over the 4-bit cache.
//
// With keys k_j = s_jg n_jd and values v_j = s_jg n_jd (g a group of 32 dims, n whole numbers), the
// scores are q . k_j = sum_g s_jg (sum_{d in g} q_d n_jd) and the result o_d = sum_j (p_j s_jg) n_jd. The
// whole numbers enter the tensor cores as they are, exact in 16 bits, positions on the MMA's 16 rows and
// query columns (rows x grouped heads, 8 to an MMA) on its 8 columns; scales meet the keys' sums in
// fp32, and the softmax weights before those go to the values' product. So the cache is read once for
// all columns of a block, and unpacked once.
//
// Bound by HBM, and close behind it by instruction issue: 4.5 bits a value arrive at 44 values per
// clock and SM, and a value takes some two instructions (unpack, product, scale).
// mma.sync and not tcgen05: its operands come from registers, where the unpacked values are; for
// tcgen05 each would have to be written to shared memory once more for at most 16 columns.
//
// Work: pieces of a (sequence, key/value head, block of columns), cut where a sequence is long, so that
// the SMs fill whatever the lengths are, which only the device knows. A warp of a piece takes every
// sixth tile of 32 positions through a ring of its own (TMA: values swizzled so that fragments
// read without bank conflicts), with a running maximum and sum; the warps join in shared memory, the
// pieces of a sequence in a second launch.
#include <cuda.h>

#include "kv4.cuh"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {
using namespace sm100;

constexpr int kWarps = 6, kThreads = kWarps * 32;
constexpr int kTok = 32;                 // positions of a tile
constexpr int kLeast = 2 * kWarps;       // tiles of a piece, where its sequence has as many
constexpr int kSlots = 2 * 148;          // pieces at a time
constexpr int kMost = 3 * kSlots;        // pieces of about even length that all work is cut into

struct Args {
  Kv4 c;
  const void* q;
  void* out;
  int64_t q_seq, q_row, q_head, o_seq, o_row, o_head;
  int window, rows, heads, group, columns, blocks;    // columns = rows x group, in `blocks` blocks
  const int32_t* pos;
  int32_t* err;
  float scale;                           // scaling log2(e)
  float *part, *ml;                      // pieces: unnormalised results [piece][column][hd]; maximum and sum
};

struct Maps {
  CUtensorMap k, v;
};

// The positions that some row of sequence b sees, in tiles.
struct Reach {
  int first, tiles;
};
__device__ __forceinline__ Reach reach_of(const Args& a, int b) {
  const int64_t p = __ldg(a.pos + b);
  const int64_t hi = min(p + a.rows, (int64_t)a.c.positions);
  const int64_t lo = a.window > 0 ? max(p + 1 - a.window, (int64_t)0) : 0;
  if (hi <= lo) return {0, 0};
  return {(int)(lo / kTok), (int)((hi + kTok - 1) / kTok - lo / kTok)};
}

// All pieces: sequence by sequence, each cut into the same number of parts for all its heads and blocks.
struct Cut {
  int parts, first_piece;
};
__device__ __forceinline__ int parts_of(int tiles, int chunk) { return tiles <= chunk ? 1 : (tiles + chunk - 1) / chunk; }

// The tiles of a piece at most, by this warp.
__device__ __forceinline__ int chunk_of(const Args& a) {
  const int lane = threadIdx.x & 31;
  int64_t total = 0;
  for (int b = lane; b < a.c.seqs; b += 32) total += reach_of(a, b).tiles;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= a.c.nkv * a.blocks;
  const int64_t even = (total + kMost - 1) / kMost;
  return (int)max(even, (int64_t)kLeast);
}

// The piece `index`: its sequence, head, block of columns and part; false past the last.
struct Piece {
  int b, head, block, part, parts;
};
__device__ __forceinline__ bool find_piece(const Args& a, int chunk, int index, Piece& r) {
  const int lane = threadIdx.x & 31;
  const int per = a.c.nkv * a.blocks;
  int64_t before = 0;
  for (int b0 = 0; b0 < a.c.seqs; b0 += 32) {
    const int b = b0 + lane;
    const int parts = b < a.c.seqs ? parts_of(reach_of(a, b).tiles, chunk) : 0;
    int sum = parts;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int64_t from = before + (int64_t)(sum - parts) * per;
    const uint32_t who = __ballot_sync(0xffffffffu, index >= from && index < from + (int64_t)parts * per);
    if (who) {
      const int src = __ffs(who) - 1;
      const int rest = __shfl_sync(0xffffffffu, (int)(index - from), src);
      r.parts = __shfl_sync(0xffffffffu, parts, src);
      r.b = b0 + src;
      r.part = rest % r.parts;
      r.block = rest / r.parts % a.blocks;
      r.head = rest / r.parts / a.blocks;
      return true;
    }
    before += (int64_t)__shfl_sync(0xffffffffu, sum, 31) * per;
  }
  return false;
}

template <int NG, int NT, typename T>
struct Cfg {
  static constexpr int kValues = kTok * 16 * NG, kScales = kTok * 2 * NG;       // bytes of a tile, keys or values
  static constexpr int kEntry = kValues + kScales;          // keys and values of a tile are entries of their own
  static constexpr int kFrag = NT * NG * 32 * 16;                               // queries as fragments
  static constexpr int kInit = std::is_same<T, __half>::value ? 0 : NT * NG * 4 * 16;
  // two CTAs an SM (227 KB of shared memory, 1 KB of it a CTA's own)
  static constexpr int kRoom = 115712 - 1024 - kFrag - kInit - 256;
  static constexpr int kFit = kRoom / (kWarps * kEntry);
  static constexpr int kDepth = kFit > 8 ? 8 : kFit;
  static constexpr int kRing = kWarps * kDepth * kEntry;
  static constexpr int kJoin = (kWarps * 8 * NT * (32 * NG + 4) + kWarps * 8 * NT * 2) * 4;      // where the warps join
  static constexpr int kSmem = 1024 + (kRing > kJoin ? kRing : kJoin) + kFrag + kInit;
  static_assert(kDepth >= 3, "keys, values and the next keys");
  static_assert(kSmem <= 232448 - 512, "shared memory of a CTA");
  static constexpr int kMask = NG == 8 ? 7 : NG == 4 ? 3 : NG == 2 ? 1 : 0;     // swizzle: 16-byte piece ^ 128-byte line
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* err) {
  for (uint32_t it = 0; it < (1u << 16); ++it) {
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if ((it & 15) == 15 && *abort) return false;
  }
  *abort = 1;
  atomicExch(err, 48);
  return false;
}
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity) {
  for (uint32_t it = 0; it < (1u << 14); ++it)
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return;
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4],
                                    const __nv_bfloat16*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4],
                                    const __half*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(r) : "r"(at));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a & mask | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}
__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Nibbles (i, i + 4) of a word, i = 0..3, as bf16 pairs 128 + nibble: the nibble in the mantissa of 128.
__device__ __forceinline__ void pairs_128(uint32_t w, uint32_t (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = and_or(w >> (4 * i), 0x000F000Fu, 0x43004300u);
}
// The same as whole numbers nibble - 8 (exact differences), in bf16 or fp16. fp16's mantissa takes a
// nibble in its first four bits (1024 + n) and in the next four (1024 + 16 n).
__device__ __forceinline__ void pairs(uint32_t w, uint32_t (&x)[4], const __nv_bfloat16*) {
  pairs_128(w, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = sub_bf2(x[i], 0x43084308u);        // 136
}
__device__ __forceinline__ void pairs(uint32_t w, uint32_t (&x)[4], const __half*) {
  const uint32_t h = w >> 8;
  const uint32_t lo[2] = {and_or(w, 0x000F000Fu, 0x64006400u), and_or(h, 0x000F000Fu, 0x64006400u)};
  const uint32_t hi[2] = {and_or(w, 0x00F000F0u, 0x64006400u), and_or(h, 0x00F000F0u, 0x64006400u)};
  const __half2 b = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));          // 1032
  const __half2 m = __halves2half2(__ushort_as_half(0x2C00), __ushort_as_half(0x2C00));          // 1 / 16
  const __half2 c = __halves2half2(__ushort_as_half(0xD480), __ushort_as_half(0xD480));          // -72
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&lo[i]), b);
    const __half2 u = __hfma2(*reinterpret_cast<const __half2*>(&hi[i]), m, c);
    x[2 * i] = *reinterpret_cast<const uint32_t*>(&l);
    x[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&u);
  }
}
__device__ __forceinline__ uint32_t pack_bf(float a, float b) {
  const __nv_bfloat162 h = __float22bfloat162_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float lo_bf(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// The scales of a position's groups.
template <int NG>
__device__ __forceinline__ void load_scales(uint32_t at, uint32_t (&w)[(NG + 1) / 2]) {
  if constexpr (NG == 8) {
    const uint4 u = lds128(at);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (NG % 2 == 0) {
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) w[i] = lds32(at + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < (NG + 1) / 2; ++i) {
      uint16_t a, b = 0;
      asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(a) : "r"(at + 4 * i));
      if (2 * i + 1 < NG) asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(b) : "r"(at + 4 * i + 2));
      w[i] = a | (uint32_t)b << 16;
    }
  }
}

template <int NG, int NT, typename T>
__global__ void __launch_bounds__(kThreads, NG * NT > 8 ? 1 : 2) kv4_attn_kernel(const Args a, const __grid_constant__ Maps M) {
  using C = Cfg<NG, NT, T>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[kWarps * C::kDepth];
  __shared__ int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* frag = smem + (C::kRing > C::kJoin ? C::kRing : C::kJoin);
  uint8_t* init = frag + C::kFrag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int hd = a.c.hd;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * C::kDepth; ++i) mbar_init(&bars[i], 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  pdl_prologue();
  const int chunk = chunk_of(a);
  Piece pc;
  if (!find_piece(a, chunk, blockIdx.x, pc)) return;
  const Reach reach = reach_of(a, pc.b);
  const int64_t pos = __ldg(a.pos + pc.b);
  const int t0 = reach.first + (int)((int64_t)reach.tiles * pc.part / pc.parts);
  const int t1 = reach.first + (int)((int64_t)reach.tiles * (pc.part + 1) / pc.parts);
  const int mine = t1 - t0 > warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;       // this warp's tiles
  __syncthreads();                                    // the barriers are there

  // a warp's ring: the values of all entries first (swizzled rows), then their scales; entry 2 i holds the
  // keys of the warp's tile i, entry 2 i + 1 its values
  uint64_t* bar = bars + warp * C::kDepth;
  uint8_t* const ring = smem + warp * C::kDepth * C::kValues;
  uint8_t* const ring_s = smem + kWarps * C::kDepth * C::kValues + warp * C::kDepth * C::kScales;
  const int64_t row0 = a.c.at(pc.b, pc.head, 0);
  const auto load = [&](int e) {                      // lane 0
    const int slot = e % C::kDepth;
    const int64_t row = row0 + (int64_t)(t0 + warp + (e >> 1) * kWarps) * kTok;
    mbar_arrive_expect_tx(&bar[slot], C::kEntry);
    tma_2d_g2s(ring + slot * C::kValues, e & 1 ? &M.v : &M.k, 0, (int)row, &bar[slot]);
    bulk_g2s(ring_s + slot * C::kScales, (e & 1 ? a.c.vs : a.c.ks) + row * NG, C::kScales, &bar[slot]);
  };
  if (lane == 0)
    for (int e = 0; e < min(2 * mine, C::kDepth); ++e) load(e);

  // the queries as the MMA's column operand: of group j, lane (g, t) holds column g's values 8 t + (0, 4),
  // (1, 5), (2, 6), (3, 7); bf16 also what 128 + nibble - n adds to a group's sum, -136 sum q
  for (int i = warp; i < NT * NG; i += kWarps) {
    const int j = i % NG, col = pc.block * 8 * NT + i / NG * 8 + g, d = 32 * j + 8 * t;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (col < a.columns && d < hd)
      x = *reinterpret_cast<const uint4*>((const T*)a.q + pc.b * a.q_seq + col / a.group * a.q_row +
                                          (pc.head * a.group + col % a.group) * a.q_head + d);
    reinterpret_cast<uint4*>(frag)[i * 32 + lane] =
        make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                   __byte_perm(x.y, x.w, 0x7632));
    if constexpr (!kHalf) {
      float s = lo_bf(x.x) + hi_bf(x.x) + lo_bf(x.y) + hi_bf(x.y) + lo_bf(x.z) + hi_bf(x.z) + lo_bf(x.w) + hi_bf(x.w);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if ((t & 1) == 0) reinterpret_cast<float*>(init)[(i * 4 + g / 2) * 4 + (g & 1) + t] = -136.f * s;   // twice
    }
  }
  __syncthreads();

  // this lane's columns (of the values' product): 8 nt + g
  int at_c[NT], low_c[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = pc.block * 8 * NT + 8 * n + g;
    const int64_t p = pos + col / a.group;
    const bool in = col < a.columns && p >= 0 && p < a.c.positions;
    at_c[n] = in ? (int)p : -1;
    low_c[n] = in && a.window > 0 ? (int)max(p + 1 - a.window, (int64_t)0) : 0;
  }
  // every column of a row sees all of positions all_low .. all_high
  const int all_high = (int)min(max(pos, (int64_t)-1), (int64_t)a.c.positions);
  const int64_t newest = min(pos + a.rows - 1, (int64_t)a.c.positions - 1);
  const int all_low = a.window > 0 ? (int)max(newest + 1 - a.window, (int64_t)0) : 0;

  float o[NG][2][NT][4];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][h][n][e] = 0.f;
  }
  // fragments' addresses in a tile: keys (row g, word t), values (row t, word g / 2)
  const uint32_t at_k = g * 16 * NG + (C::kMask ? ((g * 16 * NG >> 7) & C::kMask) << 4 : 0) + t * 4;
  const uint32_t at_v = t * 16 * NG + (C::kMask ? ((t * 16 * NG >> 7) & C::kMask) << 4 : 0) + (g >> 1) * 4;
  const uint32_t half = (g & 1) ? 0x7632 : 0x5410;    // which half of a word: 4 of its 8 dims

  int done = 0;                                       // entries
#pragma unroll 1
  for (; done < 2 * mine; ++done) {
    const int slot_k = done % C::kDepth, slot_v = (done + 1) % C::kDepth;
    if (!__all_sync(0xffffffffu, wait(&bar[slot_k], (uint32_t)(done / C::kDepth) & 1, &abort_flag, a.err))) break;
    const uint32_t ks = smem_u32(ring) + slot_k * C::kValues, vs = smem_u32(ring) + slot_v * C::kValues;
    const uint32_t kss = smem_u32(ring_s) + slot_k * C::kScales, vss = smem_u32(ring_s) + slot_v * C::kScales;
    const int p0 = (t0 + warp + (done >> 1) * kWarps) * kTok;

    // scores of 32 positions: rows g and g + 8 of two MMA tiles, columns 2 t and 2 t + 1
    float s[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[h][n][e] = 0.f;
    {
      uint32_t sc[4][(NG + 1) / 2];                   // rows g, g + 8, g + 16, g + 24
#pragma unroll
      for (int r = 0; r < 4; ++r) load_scales<NG>(kss + (g + 8 * r) * 2 * NG, sc[r]);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint32_t x[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // 8 rows are whole turns of the swizzle where there is one
          const uint32_t w = lds32(ks + (C::kMask ? at_k ^ (j << 4) : at_k + (j << 4)) + r * 128 * NG);
          if constexpr (kHalf) pairs(w, x[r], (const T*)nullptr);
          else pairs_128(w, x[r]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 q = lds128(smem_u32(frag) + ((n * NG + j) * 32 + lane) * 16);
          float zero[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (!kHalf) {
            const uint4 c = lds128(smem_u32(init) + ((n * NG + j) * 4 + t) * 16);
            zero[0] = __uint_as_float(c.x), zero[1] = __uint_as_float(c.y);
            zero[2] = __uint_as_float(c.z), zero[3] = __uint_as_float(c.w);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float d[4];
            const uint32_t a0[4] = {x[2 * h][0], x[2 * h + 1][0], x[2 * h][1], x[2 * h + 1][1]};
            const uint32_t a1[4] = {x[2 * h][2], x[2 * h + 1][2], x[2 * h][3], x[2 * h + 1][3]};
            mma(d, a0, q.x, q.y, zero, (const T*)nullptr);
            mma(d, a1, q.z, q.w, d, (const T*)nullptr);
            const float s0 = j & 1 ? hi_bf(sc[2 * h][j / 2]) : lo_bf(sc[2 * h][j / 2]);
            const float s1 = j & 1 ? hi_bf(sc[2 * h + 1][j / 2]) : lo_bf(sc[2 * h + 1][j / 2]);
            s[h][n][0] = fmaf(s0, d[0], s[h][n][0]);
            s[h][n][1] = fmaf(s0, d[1], s[h][n][1]);
            s[h][n][2] = fmaf(s1, d[2], s[h][n][2]);
            s[h][n][3] = fmaf(s1, d[3], s[h][n][3]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && done + C::kDepth < 2 * mine) load(done + C::kDepth);
    // turned: this lane's column g, positions t, t + 4, t + 8, t + 12 of each half
    float p[2][NT][4];
    const int src = t * 4 + (g >> 1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {                 // position t + 4 e: row t + 4 (e & 1) of half e / 2
          const float even = __shfl_sync(0xffffffffu, s[h][n][2 * (e >> 1)], src + 16 * (e & 1));
          const float odd = __shfl_sync(0xffffffffu, s[h][n][2 * (e >> 1) + 1], src + 16 * (e & 1));
          p[h][n][e] = (g & 1 ? odd : even) * a.scale;
        }
    const bool cut = p0 + kTok - 1 > all_high || p0 < all_low;
    if (cut) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = p0 + 16 * h + t + 4 * e;
            if (at > at_c[n] || at < low_c[n]) p[h][n][e] = -INFINITY;
          }
    }
    bool moved = false;
    float f[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = m[n];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, p[h][n][e]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      moved |= top != m[n];
      f[n] = m[n] == -INFINITY ? 0.f : ex2(m[n] - top);
      m[n] = top;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        l[n] *= f[n];
        const float f0 = __shfl_sync(0xffffffffu, f[n], 8 * t), f1 = __shfl_sync(0xffffffffu, f[n], 8 * t + 4);
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) o[j][h][n][0] *= f0, o[j][h][n][1] *= f1, o[j][h][n][2] *= f0, o[j][h][n][3] *= f1;
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float less = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[h][n][e] = ex2(p[h][n][e] - less);
          l[n] += p[h][n][e];
        }
    }

    ++done;
    if (!__all_sync(0xffffffffu, wait(&bar[slot_v], (uint32_t)(done / C::kDepth) & 1, &abort_flag, a.err))) break;
    // O += (p s) n, 16 positions at a time: k index 2 t, 2 t + 1, 2 t + 8, 2 t + 9 are positions t, t + 4, t + 8, t + 12
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t sc[4][(NG + 1) / 2];
#pragma unroll
      for (int e = 0; e < 4; ++e) load_scales<NG>(vss + (16 * h + t + 4 * e) * 2 * NG, sc[e]);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint32_t u[2], x[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // rows 4 further: half a turn of the swizzle
          const uint32_t turn = C::kMask ? ((4 * 16 * NG >> 7) & C::kMask) << 4 : 0;
          const uint32_t w0 = lds32(vs + (C::kMask ? at_v ^ (j << 4) : at_v + (j << 4)) + (16 * h + 8 * i) * 16 * NG);
          const uint32_t w1 = lds32(vs + (C::kMask ? at_v ^ (j << 4) ^ turn : at_v + (j << 4)) + (16 * h + 8 * i + 4) * 16 * NG);
          u[i] = __byte_perm(w0, w1, half);
          pairs(u[i], x[i], (const __nv_bfloat16*)nullptr);
        }
        const uint32_t a0[4] = {x[0][0], x[0][1], x[1][0], x[1][1]};
        const uint32_t a1[4] = {x[0][2], x[0][3], x[1][2], x[1][3]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float sv = j & 1 ? hi_bf(sc[e][j / 2]) : lo_bf(sc[e][j / 2]);
            if (cut) {                                // a position that this column does not see may have any scale
              const int at = p0 + 16 * h + t + 4 * e;
              if (at > at_c[n] || at < low_c[n]) sv = 0.f;
            }
            w[e] = p[h][n][e] * sv;
          }
          const uint32_t b0 = pack_bf(w[0], w[1]), b1 = pack_bf(w[2], w[3]);
          mma(o[j][0][n], a0, b0, b1, o[j][0][n], (const __nv_bfloat16*)nullptr);
          mma(o[j][1][n], a1, b0, b1, o[j][1][n], (const __nv_bfloat16*)nullptr);
          if constexpr (kHalf) {                      // what the rounding of the weights left
            const uint32_t r0 = pack_bf(w[0] - lo_bf(b0), w[1] - hi_bf(b0)), r1 = pack_bf(w[2] - lo_bf(b1), w[3] - hi_bf(b1));
            mma(o[j][0][n], a0, r0, r1, o[j][0][n], (const __nv_bfloat16*)nullptr);
            mma(o[j][1][n], a1, r0, r1, o[j][1][n], (const __nv_bfloat16*)nullptr);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && done + C::kDepth < 2 * mine) load(done + C::kDepth);
  }
  if (done < 2 * mine && lane == 0)                   // a wait gave up: the loads in flight land first
    for (int e = done; e < min(done + C::kDepth, 2 * mine); ++e) settle(&bar[e % C::kDepth], (uint32_t)(e / C::kDepth) & 1);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
  }
  __syncthreads();                                    // all tiles are read: their place is free

  // the warps join: each to the common maximum, then a thread adds a column's dims
  constexpr int kRow = 32 * NG + 4;
  float* jo = reinterpret_cast<float*>(smem);         // [warp][column][kRow]
  float* jm = jo + kWarps * 8 * NT * kRow;            // [warp][column][2]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (t == 0) {
      jm[(warp * 8 * NT + 8 * n + g) * 2] = m[n];
      jm[(warp * 8 * NT + 8 * n + g) * 2 + 1] = l[n];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {                     // columns 2 t, 2 t + 1
      float* to = jo + (warp * 8 * NT + 8 * n + 2 * t + e) * kRow + 4 * g;
      if (pc.block * 8 * NT + 8 * n + 2 * t + e < a.columns) {
#pragma unroll
        for (int j = 0; j < NG; ++j)
          *reinterpret_cast<float4*>(to + 32 * j) =
              make_float4(o[j][0][n][e], o[j][0][n][e + 2], o[j][1][n][e], o[j][1][n][e + 2]);
      }
    }
  }
  __syncthreads();
  const int per = hd / 4;
  for (int i = threadIdx.x; i < 8 * NT * per; i += kThreads) {
    const int c = i / per, d = (i - c * per) * 4, col = pc.block * 8 * NT + c;
    if (col >= a.columns) break;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, jm[(w * 8 * NT + c) * 2]);
    float L = 0.f;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = jm[(w * 8 * NT + c) * 2];
      const float4 x = *reinterpret_cast<const float4*>(jo + (w * 8 * NT + c) * kRow + d);
      const float lw = jm[(w * 8 * NT + c) * 2 + 1];
      const float fw = mw == -INFINITY ? (lw == 0.f ? 0.f : lw) : ex2(mw - M);       // NaN stays
      L += lw * fw;
      r.x += x.x * fw, r.y += x.y * fw, r.z += x.z * fw, r.w += x.w * fw;
    }
    if (pc.parts > 1) {
      const int64_t to = (int64_t)blockIdx.x * (8 * NT) + c;
      *reinterpret_cast<float4*>(a.part + to * hd + d) = r;
      if (d == 0) a.ml[to * 2] = M, a.ml[to * 2 + 1] = L;
    } else {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int64_t row = col / a.group;
      T* to = (T*)a.out + pc.b * a.o_seq + row * a.o_row + (pc.head * a.group + col % a.group) * a.o_head + d;
      const int64_t at = pos + row;
      if (at < 0 || at >= a.c.positions) {
        r = make_float4(0.f, 0.f, 0.f, 0.f);
        atomicExch(a.err, 2);
      }
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 0, r.x * inv);
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 1, r.y * inv);
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 2, r.z * inv);
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 3, r.w * inv);
    }
  }
}

// Joins the parts of sequences that were cut; a warp per column.
template <typename T>
__global__ void __launch_bounds__(256) kv4_join_kernel(const Args a, int block_columns) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);         // (sequence, head, column)
  const int64_t per_seq = (int64_t)a.c.nkv * a.columns;
  if (w >= per_seq * a.c.seqs) return;
  const int b = (int)(w / per_seq), rest = (int)(w - b * per_seq), head = rest / a.columns, col = rest % a.columns;
  const int chunk = chunk_of(a);
  const int parts = parts_of(reach_of(a, b).tiles, chunk);
  if (parts == 1) return;
  int64_t before = 0;
  for (int i = lane; i < b; i += 32) before += parts_of(reach_of(a, i).tiles, chunk);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const int64_t piece = before * a.c.nkv * a.blocks + ((int64_t)head * a.blocks + col / block_columns) * parts;
  const int64_t from = piece * block_columns + col % block_columns;
  float M = -INFINITY, L = 0.f, r[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < parts; ++i) M = fmaxf(M, a.ml[(from + (int64_t)i * block_columns) * 2]);
  for (int i = 0; i < parts; ++i) {
    const int64_t at = from + (int64_t)i * block_columns;
    const float m = a.ml[at * 2], l = a.ml[at * 2 + 1];
    const float f = m == -INFINITY ? (l == 0.f ? 0.f : l) : ex2(m - M);
    L += l * f;
    if (lane * 8 < a.c.hd) {
      const float4 x = *reinterpret_cast<const float4*>(a.part + at * a.c.hd + lane * 8);
      const float4 y = *reinterpret_cast<const float4*>(a.part + at * a.c.hd + lane * 8 + 4);
      r[0] += x.x * f, r[1] += x.y * f, r[2] += x.z * f, r[3] += x.w * f;
      r[4] += y.x * f, r[5] += y.y * f, r[6] += y.z * f, r[7] += y.w * f;
    }
  }
  const int row = col / a.group;
  const int64_t at = (int64_t)__ldg(a.pos + b) + row;
  float inv = L == 0.f ? 0.f : 1.f / L;
  const bool in = at >= 0 && at < a.c.positions;
  if (!in && lane == 0) atomicExch(a.err, 2);
  T* to = (T*)a.out + b * a.o_seq + row * a.o_row + (int64_t)(head * a.group + col % a.group) * a.o_head + lane * 8;
  if (lane * 8 < a.c.hd)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      store_from_float(to, std::is_same<T, __half>::value ? FBFP_F16 : FBFP_BF16, i, in ? r[i] * inv : 0.f);
}

// Columns that a block holds: more let one unpacking serve more columns, as far as the accumulators
// (32 registers for each 8 columns of 128 dims) leave two CTAs an SM.
int column_tiles(int64_t columns, int groups) {
  if (columns <= 8) return 1;
  if (columns <= 16 || groups > 4) return 2;
  return 4;
}

struct Plan {
  int nt, blocks;
  int64_t pieces;
  bool joins;
};
Plan plan_of(const Kv4& c, int64_t rows, int64_t heads, int64_t window) {
  Plan p;
  const int64_t columns = rows * (heads / c.nkv);
  p.nt = column_tiles(columns, c.groups);
  p.blocks = (int)((columns + 8 * p.nt - 1) / (8 * p.nt));
  const int64_t items = (int64_t)c.seqs * c.nkv * p.blocks;
  int64_t tiles = c.positions / kTok;                     // of a sequence at most
  if (window > 0 && (window + rows + kTok - 2) / kTok + 1 < tiles) tiles = (window + rows + kTok - 2) / kTok + 1;
  p.joins = tiles > kLeast;
  // parts_of adds at most one part to tiles / chunk, and all tiles / chunk are kMost at most
  p.pieces = items + (p.joins ? (items * tiles < kMost * (int64_t)kLeast ? items * tiles / kLeast : kMost) : 0);
  return p;
}

template <int NG, int NT, typename T>
int launch(const Args& a, const Maps& m, const Plan& p, cudaStream_t st) {
  auto kernel = kv4_attn_kernel<NG, NT, T>;
  static bool set[64];
  int dev = 0;
  FBFP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NG, NT, T>::kSmem));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  FBFP_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)p.pieces), dim3(kThreads), (size_t)Cfg<NG, NT, T>::kSmem, st, a, m));
  FBFP_LAUNCH_CHECK("kv4_attn_kernel");
  if (p.joins) {
    const int64_t warps = (int64_t)a.c.seqs * a.c.nkv * a.columns;
    FBFP_CUDA_TRY(launch_pdl(kv4_join_kernel<T>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, st, a, 8 * NT));
    FBFP_LAUNCH_CHECK("kv4_join_kernel");
  }
  return FBFP_OK;
}
template <int NG, typename T>
int launch_nt(const Args& a, const Maps& m, const Plan& p, cudaStream_t st) {
  if constexpr (NG <= 4)
    if (p.nt == 4) return launch<NG, 4, T>(a, m, p, st);
  return p.nt == 1 ? launch<NG, 1, T>(a, m, p, st) : launch<NG, 2, T>(a, m, p, st);
}
template <typename T>
int launch_ng(const Args& a, const Maps& m, const Plan& p, cudaStream_t st) {
  switch (a.c.groups) {
    case 1: return launch_nt<1, T>(a, m, p, st);
    case 2: return launch_nt<2, T>(a, m, p, st);
    case 3: return launch_nt<3, T>(a, m, p, st);
    case 4: return launch_nt<4, T>(a, m, p, st);
    case 5: return launch_nt<5, T>(a, m, p, st);
    case 6: return launch_nt<6, T>(a, m, p, st);
    case 7: return launch_nt<7, T>(a, m, p, st);
    default: return launch_nt<8, T>(a, m, p, st);
  }
}

}  // namespace
}  // namespace fbfp

using namespace fbfp;

extern "C" int64_t fbfp_kv4_attention_workspace_bytes(const fbfp_kv4_cache* cache, int64_t rows, int64_t heads) {
  Kv4 c;
  if (kv4_check(cache, c) || rows < 1 || heads < 1 || heads % c.nkv) return -1;
  const Plan p = plan_of(c, rows, heads, 0);
  return p.joins ? p.pieces * 8 * p.nt * (c.hd + 2) * 4 : 0;
}

extern "C" int fbfp_kv4_attention(const fbfp_kv4_cache* cache, const void* q, int dtype, int64_t rows, int64_t heads,
                                  int64_t q_seq, int64_t q_row, int64_t q_head, const int32_t* pos, int64_t window,
                                  float scaling, void* out, int64_t o_seq, int64_t o_row, int64_t o_head,
                                  void* workspace, int64_t workspace_bytes, int32_t* err, void* stream) {
  Kv4 c;
  int st = kv4_check(cache, c);
  if (st) return st;
  FBFP_CHECK_ARG(q && pos && out && err, "null pointer");
  FBFP_CHECK_ARG(dtype == FBFP_BF16 || dtype == FBFP_F16, "bad dtype %d (bf16 or fp16)", dtype);
  FBFP_CHECK_ARG(rows >= 1 && rows <= 65535 && heads >= 1 && heads <= 65535 && heads % c.nkv == 0,
                 "bad rows %lld, or %lld heads over %d", (long long)rows, (long long)heads, c.nkv);
  FBFP_CHECK_ARG(q_seq >= 0 && q_row >= 0 && q_head >= 0 && o_seq >= 0 && o_row >= 0 && o_head >= 0 &&
                     ((q_seq | q_row | q_head | o_seq | o_row | o_head) & 7) == 0,
                 "strides must be multiples of 8");
  FBFP_CHECK_ARG(window >= 0, "negative window");
  if (((uintptr_t)q | (uintptr_t)out) & 15) return set_error(FBFP_ERR_ALIGN, "q and out must be 16-byte aligned");
  FBFP_CHECK_ARG((int64_t)c.seqs * c.nkv * c.positions < ((int64_t)1 << 31), "the cache has 2^31 rows or more");
  if (window > c.positions + rows) window = 0;              // sees everything
  const Plan p = plan_of(c, rows, heads, window);
  FBFP_CHECK_ARG(p.pieces <= 0x7FFFFFFF && (int64_t)c.seqs * heads * rows < ((int64_t)1 << 31), "too many rows");
  const int64_t need = p.joins ? p.pieces * 8 * p.nt * (c.hd + 2) * 4 : 0;
  FBFP_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                 "the workspace must be %lld bytes, 16-byte aligned", (long long)need);
  const int group = (int)(heads / c.nkv);
  Args a{c, q, out, q_seq, q_row, q_head, o_seq, o_row, o_head, (int)window, (int)rows, (int)heads, group,
         (int)rows * group, p.blocks, pos, err, scaling * 1.4426950408889634f, (float*)workspace,
         (float*)workspace + p.pieces * 8 * p.nt * c.hd};
  Maps m;
  const uint64_t cells = (uint64_t)c.seqs * c.nkv * c.positions;
  const CUtensorMapSwizzle swz = c.groups == 8   ? CU_TENSOR_MAP_SWIZZLE_128B
                                 : c.groups == 4 ? CU_TENSOR_MAP_SWIZZLE_64B
                                 : c.groups == 2 ? CU_TENSOR_MAP_SWIZZLE_32B
                                                 : CU_TENSOR_MAP_SWIZZLE_NONE;
  st = encode_2d(&m.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.kv, 16 * c.groups, cells, 16 * c.groups, 16 * c.groups, kTok, swz);
  if (!st) st = encode_2d(&m.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.vv, 16 * c.groups, cells, 16 * c.groups, 16 * c.groups, kTok, swz);
  if (st) return st;
  return dtype == FBFP_BF16 ? launch_ng<__nv_bfloat16>(a, m, p, as_stream(stream)) : launch_ng<__half>(a, m, p, as_stream(stream));
}
