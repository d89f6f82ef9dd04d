// kv4_attn.cu — attention of the newest rows of each sequence over the 4-bit cache.
//
// With keys k_j = s_jg n_jd and values v_j = s_jg n_jd (g a group of 32 dims, n whole numbers), the
// scores are q . k_j = sum_g s_jg (sum_{d in g} q_d n_jd) and the result o_d = sum_j (p_j s_jg) n_jd. The
// whole numbers enter the tensor cores as they are, exact in 16 bits, positions on the MMA's 16 rows and
// query columns (rows x grouped heads, 8 to an MMA) on its 8 columns; scales meet the keys' sums in
// fp32, and the softmax weights before those go to the values' product. So the cache is read once for
// all columns of a block, and unpacked once.
//
// Bound by the latency of dependent instructions in twelve warps an SM: a warp takes some 1300 instructions for a
// tile of 32 positions x 256 values (unpack, products, scales), of which 2.5 issue in a clock and SM (58% of the
// slots, the integer pipe busy half the time), and 168 registers a thread leave no room for more warps; the loads
// alone take two thirds as long. 16 sequences of 9000 to 32700 positions, 8 heads of 256 for 16 query heads: 175-177
// us, 3.9 TB/s. 64 sequences of 500 to 8100 positions with 4 rows each, 64 query heads on 8 of 128: 250 us,
// where the unpacked values meet 32 columns in two blocks of 16 and the softmax of those counts as much.
// mma.sync and not tcgen05: its operands come from registers, where the unpacked values are; for
// tcgen05 each would have to be written to shared memory once more for at most 16 columns.
//
// Work: all tiles of 32 positions in one list, of which each CTA takes an even share, so that the SMs fill
// and end together whatever the lengths are, which only the device knows. A warp takes every sixth (twelfth) tile
// through a ring of its own (TMA: values swizzled so that fragments read without bank conflicts),
// with a running maximum and sum; the warps join in shared memory, parts of a sequence in a second
// launch.
#include <cuda.h>
#include <cmath>

#include "kv4.cuh"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {
using namespace sm100;

constexpr int kTok = 32;                 // positions of a tile
constexpr int kLeast = 12;               // tiles that are worth a CTA
constexpr int kSms = 148;
constexpr int kAccumulators = 8;         // 32 dims x 8 columns each, of a warp at most: 64 registers of a thread

struct Args {
  Kv4 c;
  const void* q;
  void* out;
  int64_t q_seq, q_row, q_head, o_seq, o_row, o_head;
  int window, rows, heads, group, columns, blocks;    // columns = rows x group, in `blocks` blocks
  const int32_t* pos;
  int32_t* err;
  int slots;                             // CTAs at a time
  float scale;                           // scaling log2(e)
  float *part, *ml;                      // segments: unnormalised results [segment][column][hd]; maximum and sum
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

// All work is a list of items, (sequence, key/value head, block of columns), sequence by sequence, of
// so many tiles each (at least one, so that each item has a CTA). Where every item, cut into parts of kLeast
// tiles, fits the SMs at once, a CTA takes one part (the list is padded to whole parts); else each CTA takes the
// same length of the list, as many items or parts of items as that is. What a CTA does of one item
// is a segment; segment number = CTA + item, each its own. (A cache has fewer than 2^26 tiles, so that the list
// counts in 32 bits for up to 32 blocks of columns: the call checks.)
struct Schedule {
  bool parts;
  uint32_t share, total;                 // tiles a CTA, of all (padded)
};
__device__ __forceinline__ uint32_t padded(int tiles, bool parts) {
  const uint32_t n = max(tiles, 1);
  return parts ? (n + kLeast - 1) / kLeast * kLeast : n;
}
// By this warp. `mine`: the tiles of sequence `lane`.
__device__ __forceinline__ Schedule schedule_of(const Args& a, int& mine) {
  uint32_t total = 0, parts = 0;
  for (int b = threadIdx.x & 31; b < a.c.seqs; b += 32) {
    const int n = reach_of(a, b).tiles;
    if (b < 32) mine = n;
    total += padded(n, false);
    parts += padded(n, true) / kLeast;
  }
  const uint32_t per = a.c.nkv * a.blocks;
  total = __reduce_add_sync(0xffffffffu, total) * per;
  parts = __reduce_add_sync(0xffffffffu, parts) * per;
  if (parts <= (uint32_t)a.slots) return {true, kLeast, parts * kLeast};
  return {false, max((total + a.slots - 1) / a.slots, (uint32_t)kLeast), total};
}
// The sequence that place `at` (below the total) of the list is in, and where its first item begins.
__device__ __forceinline__ void find_sequence(const Args& a, const Schedule& s, uint32_t at, int mine, int& seq,
                                              uint32_t& begin) {
  const int lane = threadIdx.x & 31;
  const uint32_t per = a.c.nkv * a.blocks;
  uint32_t before = 0;
  for (int b0 = 0; b0 < a.c.seqs; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t n = b < a.c.seqs ? padded(b0 == 0 ? mine : reach_of(a, b).tiles, s.parts) * per : 0;
    uint32_t sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, at >= before + sum - n && at < before + sum);
    if (who) {
      const int src = __ffs(who) - 1;
      seq = b0 + src;
      begin = before + __shfl_sync(0xffffffffu, sum - n, src);
      return;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  seq = 0, begin = 0;                                 // not reached
}

struct Piece {
  int b, head, block;
};

template <int NG, int NT, int WARPS>
struct Cfg {
  // Twelve warps an SM, 168 registers a thread: two CTAs of six, one's start and end beside the other's tiles; or
  // one of twelve, where each CTA has a part of at most twelve tiles and the time is that of one tile.
  static constexpr int kWarps = WARPS, kCtas = 12 / WARPS, kThreads = kWarps * 32;
  static constexpr int kValues = kTok * 16 * NG, kScales = kTok * 2 * NG;       // bytes of a tile, keys or values
  static constexpr int kMostDepth = NG > 6 ? 4 : 8;
  static constexpr int kEntry = kValues + kScales;          // keys and values of a tile are entries of their own
  static constexpr int kFrag = NT * NG * 32 * 16;                               // queries as fragments
  static constexpr int kColumns = 8 * NT * 4;
  // of 228 KB shared memory an SM, 1 KB of it each CTA's own
  static constexpr int kMore = kFrag + kColumns + kWarps * 8 * kMostDepth + 16;  // barriers, the word that says that a wait gave up
  static constexpr int kMost = kCtas == 2 ? 115712 : 232448, kRoom = kMost - kMore;
  static constexpr int kFit = kRoom / (kWarps * kEntry);
  static constexpr int kDepth = kFit > kMostDepth ? kMostDepth : kFit;
  static constexpr int kRing = kWarps * kDepth * kEntry;
  static constexpr int kJoin = (kWarps * 8 * NT * (32 * NG + 4) + kWarps * 8 * NT * 2) * 4;      // where the warps join
  static constexpr int kSmem = (kRing > kJoin ? kRing : kJoin) + kMore;
  static_assert(kDepth >= 3, "keys, values and the next keys");
  static_assert(kSmem <= kMost, "shared memory of a CTA");
  static constexpr int kMask = NG == 8 ? 7 : NG == 4 ? 3 : NG == 2 ? 1 : 0;     // swizzle: 16-byte piece ^ 128-byte line
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* err) {
  if (mbar_wait_second(bar, parity, abort)) return true;
  *abort = 1;
  atomicExch(err, 48);
  return false;
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
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
// a & mask | 1024 in each half, in one instruction.
__device__ __forceinline__ uint32_t in_1024(uint32_t a, uint32_t mask) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, 0x64006400, 0xEA;" : "=r"(r) : "r"(a), "r"(mask));
  return r;
}
__device__ __forceinline__ uint32_t half2_fma(uint32_t a, uint32_t m, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(m), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t half2_add(uint32_t a, uint32_t c) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(c));
  return r;
}
// Nibbles n = 0..3 of each half of a word as fp16 pairs n - 8: in the first four bits of 1024's mantissa a
// nibble makes it 1024 + n, in the next four 1024 + 16 n; - 1032, or / 16 - 72, is exact. (The conversion of
// 4-bit weights by one logic operation and one of fp16 arithmetic: Kim, Henry, Fahim and Awadalla, "Who Says
// Elephants Can't Run", 2022.)
__device__ __forceinline__ void pairs(uint32_t w, uint32_t (&x)[4]) {
  const uint32_t h = w >> 8;
  x[0] = half2_add(in_1024(w, 0x000F000Fu), 0xE408E408u);
  x[1] = half2_fma(in_1024(w, 0x00F000F0u), 0x2C002C00u, 0xD480D480u);
  x[2] = half2_add(in_1024(h, 0x000F000Fu), 0xE408E408u);
  x[3] = half2_fma(in_1024(h, 0x00F000F0u), 0x2C002C00u, 0xD480D480u);
}
__device__ __forceinline__ uint32_t pack_h(float a, float b) {
  const __half2 h = __float22half2_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float lo_h(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)w)); }
__device__ __forceinline__ float hi_h(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)(w >> 16))); }
__device__ __forceinline__ void fma2(float& a0, float& a1, float x0, float x1, float y) {
  asm("{\n\t.reg .b64 a, x, y;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\t"
      "fma.rn.f32x2 a, x, y, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1) : "f"(x0), "f"(x1), "f"(y));
}
__device__ __forceinline__ void mul2(float& r0, float& r1, float x0, float x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r0), "=f"(r1) : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
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

// The bits of the largest finite scale of 32 positions' values, of those that some column of the block sees:
// a position per lane. `low`: the lane's smallest scale but 0, less one (or two) in its bits; 0xFFFF: none.
template <int NG>
__device__ __forceinline__ uint32_t largest_scale(uint32_t vss, bool counts, uint32_t& low) {
  uint32_t w[(NG + 1) / 2], high = 0, least = 0xFFFFFFFFu;              // in halves
  load_scales<NG>(vss + (threadIdx.x & 31) * 2 * NG, w);
#pragma unroll
  for (int i = 0; i < (NG + 1) / 2; ++i) high = __vmaxu2(high, w[i]), least = __vminu2(least, w[i] - 0x00010001u);
  high = counts ? max(high & 0xFFFFu, high >> 16) : 0;
  low = counts ? min(least & 0xFFFFu, least >> 16) : 0xFFFFu;
  high = __reduce_max_sync(0xffffffffu, high);
  if (high < 0x7F80u) return high;
  high = 0;                                           // infinite and NaN scales make their own dims NaN: the rest counts
#pragma unroll
  for (int i = 0; i < (NG + 1) / 2; ++i) {
    const uint32_t w0 = w[i] & 0x7FFFu, w1 = (w[i] >> 16) & 0x7FFFu;
    high = max(high, max(w0 >= 0x7F80u ? 0u : w0, w1 >= 0x7F80u ? 0u : w1));
  }
  return __reduce_max_sync(0xffffffffu, counts ? high : 0u);
}

// O += (p s) n of 32 positions. The weights p carry a power of two that brings (p s) into fp16's range: 2^15 at most,
// 2^8 where the largest weight meets the largest scale. What is below 2^-25 vanishes, which is nothing beside a
// result in which the largest weight meets a scale 2^-kDeep as large; where smaller ones were met, add_in_rounds
// takes this one's place.
// CUT: some column does not see some position, whose scale may be anything.
template <int NG, int NT, int WARPS, bool CUT>
__device__ __forceinline__ void add_values(float (&o)[NG][2][NT][4], const float (&p)[2][NT][4],
                                           uint32_t vss, uint32_t vb, uint32_t half, int p0,
                                           const int (&at_c)[NT], const int (&low_c)[NT]) {
  using C = Cfg<NG, NT, WARPS>;
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t sc[4][(NG + 1) / 2];
#pragma unroll
    for (int e = 0; e < 4; ++e) load_scales<NG>(vss + (16 * h + t + 4 * e) * 2 * NG, sc[e]);
    // k index 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of 16 positions are t, t + 4, t + 8, t + 12
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint32_t x[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        constexpr uint32_t turn = C::kMask ? ((4 * 16 * NG >> 7) & C::kMask) << 4 : 0;   // rows 4 further
        const uint32_t w0 = lds32((C::kMask ? vb ^ (j << 4) : vb + (j << 4)) + (16 * h + 8 * i) * 16 * NG);
        const uint32_t w1 = lds32((C::kMask ? vb ^ ((j << 4) ^ turn) : vb + (j << 4)) + (16 * h + 8 * i + 4) * 16 * NG);
        pairs(__byte_perm(w0, w1, half), x[i]);
      }
      const uint32_t a0[4] = {x[0][0], x[0][1], x[1][0], x[1][1]};
      const uint32_t a1[4] = {x[0][2], x[0][3], x[1][2], x[1][3]};
      float s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = j & 1 ? hi_bf(sc[e][j / 2]) : lo_bf(sc[e][j / 2]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
        if constexpr (CUT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = p0 + 16 * h + t + 4 * e;
            w[e] = at <= at_c[n] && at >= low_c[n] ? p[h][n][e] * s[e] : 0.f;
          }
        } else {
          mul2(w[0], w[1], p[h][n][0], p[h][n][1], s[0], s[1]);
          mul2(w[2], w[3], p[h][n][2], p[h][n][3], s[2], s[3]);
        }
        const uint32_t b0 = pack_h(w[0], w[1]), b1 = pack_h(w[2], w[3]);
        mma(o[j][0][n], a0, b0, b1, o[j][0][n]);
        mma(o[j][1][n], a1, b0, b1, o[j][1][n]);
      }
    }
  }
}

constexpr int kDeep = 14;
// The same in several rounds: the products from 2^-14 on, from 2^-28 on and so on, each brought up to the first one's
// range. Out of line, on copies in memory: inlined it took registers from every tile (8 sequences in a window 17.8 ->
// 21.4 us, 16 long sequences 172 -> 182). 16 sequences of 20000 positions with scales 2^16 apart in every tile: 484
// us, in one tile 192, in none 186.
template <int NG, int NT>
struct Rounds {
  float o[NG][2][NT][4], p[2][NT][4];
  int at_c[NT], low_c[NT];
};
template <int NG, int NT, int MASK>
__device__ __noinline__ void add_in_rounds(Rounds<NG, NT>& m, uint32_t vss, uint32_t vb, uint32_t half, int p0, int rounds) {
  const int t = threadIdx.x & 3;
  float p[2][NT][4];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = p0 + 16 * h + t + 4 * e;
        p[h][n][e] = at <= m.at_c[n] && at >= m.low_c[n] ? m.p[h][n][e] : -1.f;        // -1: not seen
      }
#pragma unroll 1
  for (int j = 0; j < NG; ++j) {
    float o[2][NT][4];
#pragma unroll
    for (int i = 0; i < 8 * NT; ++i) (&o[0][0][0])[i] = (&m.o[j][0][0][0])[i];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t x[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        constexpr uint32_t turn = MASK ? ((4 * 16 * NG >> 7) & MASK) << 4 : 0;                 // rows 4 further
        const uint32_t w0 = lds32((MASK ? vb ^ (j << 4) : vb + (j << 4)) + (16 * h + 8 * i) * 16 * NG);
        const uint32_t w1 = lds32((MASK ? vb ^ ((j << 4) ^ turn) : vb + (j << 4)) + (16 * h + 8 * i + 4) * 16 * NG);
        pairs(__byte_perm(w0, w1, half), x[i]);
      }
      const uint32_t a0[4] = {x[0][0], x[0][1], x[1][0], x[1][1]};
      const uint32_t a1[4] = {x[0][2], x[0][3], x[1][2], x[1][3]};
      float s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t bits;
        asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(bits) : "r"(vss + ((16 * h + t + 4 * e) * NG + j) * 2));
        s[e] = bf16_bits_to_float(bits);
      }
#pragma unroll 1
      for (int round = 0; round < rounds; ++round) {
        const float down = __uint_as_float((uint32_t)(127 - kDeep * round) << 23);
        const float up = __uint_as_float((uint32_t)(127 + kDeep * round) << 23);
        const float least = round + 1 < rounds ? down * __uint_as_float((uint32_t)(127 - kDeep) << 23) : 0.f;
        bool none = true;
        uint32_t b[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = p[h][n][e] * s[e];
            const bool mine = round == 0 ? !(y < least) : y < down && y >= least;      // (the first takes NaN)
            w[e] = p[h][n][e] != -1.f && mine ? y * up : 0.f;
          }
          b[n][0] = pack_h(w[0], w[1]), b[n][1] = pack_h(w[2], w[3]);
          none &= (b[n][0] | b[n][1]) == 0;
        }
        if (__all_sync(0xffffffffu, none)) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float zero[4] = {0.f, 0.f, 0.f, 0.f};
          float d0[4], d1[4];
          mma(d0, a0, b[n][0], b[n][1], zero);
          mma(d1, a1, b[n][0], b[n][1], zero);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[0][n][e] = fmaf(d0[e], down, o[0][n][e]), o[1][n][e] = fmaf(d1[e], down, o[1][n][e]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8 * NT; ++i) (&m.o[j][0][0][0])[i] = (&o[0][0][0])[i];
  }
}

template <int NG, int NT, int WARPS, typename T>
__global__ void __launch_bounds__((Cfg<NG, NT, WARPS>::kThreads), (Cfg<NG, NT, WARPS>::kCtas))
kv4_attn_kernel(const Args a, const __grid_constant__ Maps M) {
  using C = Cfg<NG, NT, WARPS>;
  constexpr int kWarps = C::kWarps, kThreads = C::kThreads;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem[];   // (no other shared memory in front of it)
  uint8_t* frag = smem + (C::kRing > C::kJoin ? C::kRing : C::kJoin);
  float* column_scale = reinterpret_cast<float*>(frag + C::kFrag);
  uint64_t* bars = reinterpret_cast<uint64_t*>(frag + C::kFrag + C::kColumns);
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(bars + kWarps * C::kMostDepth);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int hd = a.c.hd;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * C::kDepth; ++i) mbar_init(&bars[i], 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  pdl_prologue();
  int tiles0 = 0;                                     // of sequence `lane`
  const Schedule sch = schedule_of(a, tiles0);
  // a warp's ring: the values of all entries first (swizzled rows), then their scales; the keys and
  // the values of a tile are entries that follow each other
  uint64_t* bar = bars + warp * C::kDepth;
  uint8_t* const ring = smem + warp * C::kDepth * C::kValues;
  uint8_t* const ring_s = smem + kWarps * C::kDepth * C::kValues + warp * C::kDepth * C::kScales;
  int base = 0;                                       // entries of the segments before
  const uint32_t end = min((blockIdx.x + 1) * sch.share, sch.total);
#pragma unroll 1
  for (uint32_t at = blockIdx.x * sch.share; at < end;) {
  Piece pc;
  uint32_t begin;
  find_sequence(a, sch, at, tiles0, pc.b, begin);
  const Reach reach = reach_of(a, pc.b);
  const int64_t pos = __ldg(a.pos + pc.b);
  const uint32_t n_item = padded(reach.tiles, sch.parts);
  const uint32_t nth = (at - begin) / n_item, in_item = (at - begin) - nth * n_item;
  const int64_t item = (int64_t)pc.b * a.c.nkv * a.blocks + nth;
  pc.head = (int)(nth / a.blocks);
  pc.block = (int)(nth - pc.head * a.blocks);
  const uint32_t length = min(n_item - in_item, end - at);
  at += length;
  const bool whole = length == n_item;
  int t0, t1;                                         // tiles of the sequence
  if (sch.parts) {                                    // parts of even length
    const uint32_t parts = n_item / kLeast, part = in_item / kLeast;
    t0 = reach.first + (int)((uint64_t)reach.tiles * part / parts);
    t1 = reach.first + (int)((uint64_t)reach.tiles * (part + 1) / parts);
  } else {
    t0 = reach.first + (int)in_item;
    t1 = reach.first + min((int)(in_item + length), reach.tiles);
  }
  const int mine = t1 - t0 > warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;       // this warp's tiles
  // The queries are asked for before the tiles, which fill what is under way to memory (16 long sequences: 5.9 us
  // from here to the fragments, 3.5 this way; 64 sequences with 4 rows each 256 -> 245 us in all). With one tile of
  // columns a lane's row is the same for all its fragments.
  constexpr int kRounds = (NT * NG + kWarps - 1) / kWarps, kRows = NT == 1 ? 1 : kRounds;
  uint4 raw[kRows][NG];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int i = warp + r * kWarps, col = pc.block * 8 * NT + (NT == 1 ? 0 : i / NG * 8) + g;
    const T* row = (const T*)a.q + pc.b * a.q_seq + col / a.group * a.q_row + (pc.head * a.group + col % a.group) * a.q_head;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int d = 32 * k + 8 * t;
      raw[r][k] = make_uint4(0, 0, 0, 0);
      if (i < NT * NG && col < a.columns && d < hd) raw[r][k] = *reinterpret_cast<const uint4*>(row + d);
    }
  }
  __syncthreads();                                    // the barriers are there; the last segment's join is read
  const int64_t row0 = a.c.at(pc.b, pc.head, 0);
  const auto load = [&](int e) {                      // lane 0: entry e of the segment
    const int slot = (base + e) % C::kDepth;
    const int64_t row = row0 + (int64_t)(t0 + warp + (e >> 1) * kWarps) * kTok;
    mbar_arrive_expect_tx(&bar[slot], C::kEntry);
    tma_2d_g2s(ring + slot * C::kValues, e & 1 ? &M.v : &M.k, 0, (int)row, &bar[slot]);
    bulk_g2s(ring_s + slot * C::kScales, (e & 1 ? a.c.vs : a.c.ks) + row * NG, C::kScales, &bar[slot]);
  };
  if (lane == 0)
    for (int e = 0; e < min(2 * mine, C::kDepth); ++e) load(e);

  // the queries as the MMA's column operand: of group j, lane (g, t) holds column g's values 8 t + (0, 4),
  // (1, 5), (2, 6), (3, 7). A power of two per column brings its largest value to 2^12: bf16 values down to 2^-29
  // of the largest are exact in fp16.
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = warp + r * kWarps, j = i % NG;
    if (i >= NT * NG) break;
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const uint4 u = raw[NT == 1 ? 0 : r][k];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y0 = kHalf ? lo_h(w[e]) : lo_bf(w[e]), y1 = kHalf ? hi_h(w[e]) : hi_bf(w[e]);
        top = max(top, max(__float_as_uint(y0) & 0x7FFFFFFFu, __float_as_uint(y1) & 0x7FFFFFFFu));
        if (k == j) x[2 * e] = y0, x[2 * e + 1] = y1;
      }
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = min(max((int)(top >> 23) - 127, -100), 127);
    const float up = __uint_as_float((uint32_t)(127 + 12 - ex) << 23);
    if (j == 0 && t == 0) column_scale[i / NG * 8 + g] = a.scale * __uint_as_float((uint32_t)(ex - 12 + 127) << 23);
    reinterpret_cast<uint4*>(frag)[i * 32 + lane] = make_uint4(pack_h(x[0] * up, x[4] * up), pack_h(x[1] * up, x[5] * up),
                                                               pack_h(x[2] * up, x[6] * up), pack_h(x[3] * up, x[7] * up));
  }
  __syncthreads();

  // this lane's columns (of the values' product): 8 nt + g
  int at_c[NT], low_c[NT];
  float scale[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = pc.block * 8 * NT + 8 * n + g;
    const int64_t p = pos + col / a.group;
    const bool in = col < a.columns && p >= 0 && p < a.c.positions;
    at_c[n] = in ? (int)p : -1;
    low_c[n] = in && a.window > 0 ? (int)max(p + 1 - a.window, (int64_t)0) : 0;
    scale[n] = column_scale[8 * n + g];
  }
  // every column of a row sees all of positions all_low .. all_high
  const int all_high = (int)min(max(pos, (int64_t)-1), (int64_t)a.c.positions);
  const int64_t newest = min(pos + a.rows - 1, (int64_t)a.c.positions - 1);
  const int all_low = a.window > 0 ? (int)max(newest + 1 - a.window, (int64_t)0) : 0;

  float o[NG][2][NT][4];
  float m[NT], l[NT];
  int ev = -1000;                                     // weights are 2^(score - m + 8 - ev), ev near the scales' largest exponent
  uint32_t low = 0xFFFFu;                             // the smallest scale that this lane met
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
    const int slot_k = (base + done) % C::kDepth, slot_v = (base + done + 1) % C::kDepth;
    if (!__all_sync(0xffffffffu, wait(&bar[slot_k], (uint32_t)((base + done) / C::kDepth) & 1, &abort_flag, a.err))) break;
    const uint32_t kb = smem_u32(ring) + slot_k * C::kValues + at_k, vb = smem_u32(ring) + slot_v * C::kValues + at_v;
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
        for (int r = 0; r < 4; ++r)                   // 8 rows are whole turns of the swizzle where there is one
          pairs(lds32((C::kMask ? kb ^ (j << 4) : kb + (j << 4)) + r * 128 * NG), x[r]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 q = lds128(smem_u32(frag) + ((n * NG + j) * 32 + lane) * 16);
          const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float d[4];
            const uint32_t a0[4] = {x[2 * h][0], x[2 * h + 1][0], x[2 * h][1], x[2 * h + 1][1]};
            const uint32_t a1[4] = {x[2 * h][2], x[2 * h + 1][2], x[2 * h][3], x[2 * h + 1][3]};
            mma(d, a0, q.x, q.y, zero);
            mma(d, a1, q.z, q.w, d);
            const float s0 = j & 1 ? hi_bf(sc[2 * h][j / 2]) : lo_bf(sc[2 * h][j / 2]);
            const float s1 = j & 1 ? hi_bf(sc[2 * h + 1][j / 2]) : lo_bf(sc[2 * h + 1][j / 2]);
            if constexpr (NT == 1) {                  // a pair needs its scale twice: not worth it for one
              s[h][n][0] = fmaf(s0, d[0], s[h][n][0]), s[h][n][1] = fmaf(s0, d[1], s[h][n][1]);
              s[h][n][2] = fmaf(s1, d[2], s[h][n][2]), s[h][n][3] = fmaf(s1, d[3], s[h][n][3]);
            } else {
              fma2(s[h][n][0], s[h][n][1], d[0], d[1], s0);
              fma2(s[h][n][2], s[h][n][3], d[2], d[3], s1);
            }
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
          p[h][n][e] = (g & 1 ? odd : even) * scale[n];
        }
    ++done;
    if (!__all_sync(0xffffffffu, wait(&bar[slot_v], (uint32_t)((base + done) / C::kDepth) & 1, &abort_flag, a.err))) break;
    const bool cut = p0 + kTok - 1 > all_high || p0 < all_low;
    bool counts = true;                               // some column of the block sees position p0 + lane
    if (cut) {
      counts = p0 + lane <= newest && p0 + lane >= (a.window > 0 ? pos + 1 - a.window : 0);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at_p = p0 + 16 * h + t + 4 * e;
            if (at_p > at_c[n] || at_p < low_c[n]) p[h][n][e] = -INFINITY;
          }
    }
    uint32_t here;
    const uint32_t high = largest_scale<NG>(vss, counts, here);
    low = min(low, here);
    const int ex = min(max((int)(high >> 7) - 127, -90), 120);
    const bool grown = ex > ev + 3;                   // the references move when weights could pass 2^14 in fp16
    const float turn = grown ? (ev < -90 ? 0.f : ex2((float)(ev - ex))) : 1.f;
    if (grown) ev = ex;
    bool moved = grown;
    float f[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = p[0][n][0];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, p[h][n][e]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool raise = top > m[n] + 3.f;
      f[n] = raise ? ex2(m[n] - top) * turn : turn;   // 0 where nothing was seen yet
      if (raise) m[n] = top;
      moved |= raise;
    }
    if (__any_sync(0xffffffffu, moved) && done > 1) {
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
      const float add = (m[n] == -INFINITY ? 0.f : -m[n]) + (float)(8 - ev);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[h][n][e] = ex2(p[h][n][e] + add);
          l[n] += p[h][n][e];
        }
    }
    // Rounds, where scales met lie so far below the largest, and this tile's products reach so low.
    int rounds = 1;
    if (__any_sync(0xffffffffu, low < (uint32_t)(ev - kDeep + 127) << 7)) {
      float p_low = INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) p_low = fminf(p_low, p[h][n][e] == 0.f ? INFINITY : p[h][n][e]);
      p_low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(p_low)));
      if (!(p_low * bf16_bits_to_float(__reduce_min_sync(0xffffffffu, here)) >= __uint_as_float((uint32_t)(127 - kDeep) << 23))) {
        const uint32_t least = __reduce_min_sync(0xffffffffu, low);
        rounds = min((ev - (least < 0x80u ? -133 : (int)(least >> 7) - 127) + kDeep - 1) / kDeep, 9);
      }
    }
    if (rounds > 1) {                                 // the same in all lanes
      Rounds<NG, NT> r;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        r.at_c[n] = at_c[n], r.low_c[n] = low_c[n];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            r.p[h][n][e] = p[h][n][e];
#pragma unroll
            for (int j = 0; j < NG; ++j) r.o[j][h][n][e] = o[j][h][n][e];
          }
      }
      add_in_rounds<NG, NT, C::kMask>(r, vss, vb, half, p0, rounds);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < NG; ++j) o[j][h][n][e] = r.o[j][h][n][e];
    } else if (cut) {
      add_values<NG, NT, WARPS, true>(o, p, vss, vb, half, p0, at_c, low_c);
    } else {
      add_values<NG, NT, WARPS, false>(o, p, vss, vb, half, p0, at_c, low_c);
    }
    __syncwarp();
    if (lane == 0 && done + C::kDepth < 2 * mine) load(done + C::kDepth);
  }
  if (done < 2 * mine && lane == 0)                   // a wait gave up: the loads in flight land first
    for (int e = done; e < min(done + C::kDepth, 2 * mine); ++e) mbar_settle(&bar[(base + e) % C::kDepth], (uint32_t)((base + e) / C::kDepth) & 1);
  base += 2 * mine;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
    // sums and results are 2^(8 - ev) as large as the weights 2^(score - m) make them
    if (m[n] != -INFINITY) m[n] += (float)(ev - 8);
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
    if (!whole) {
      const int64_t to = ((int64_t)blockIdx.x + item) * (8 * NT) + c;
      *reinterpret_cast<float4*>(a.part + to * hd + d) = r;
      if (d == 0) a.ml[to * 2] = M, a.ml[to * 2 + 1] = L;
    } else {
      float inv = L == 0.f ? 0.f : 1.f / L;
      const int64_t row = col / a.group;
      T* to = (T*)a.out + pc.b * a.o_seq + row * a.o_row + (pc.head * a.group + col % a.group) * a.o_head + d;
      if (pos + row < 0 || pos + row >= a.c.positions) {              // (L may be NaN)
        r = make_float4(0.f, 0.f, 0.f, 0.f), inv = 0.f;
        atomicMax(a.err, 2);
      }
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 0, r.x * inv);
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 1, r.y * inv);
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 2, r.z * inv);
      store_from_float(to, kHalf ? FBFP_F16 : FBFP_BF16, 3, r.w * inv);
    }
  }
  fence_async_proxy();                                // the next segment's loads land where this one joined
  if (abort_flag) break;
  }
}

// Joins the segments of items that were cut; a warp per column.
template <typename T>
__global__ void __launch_bounds__(256) kv4_join_kernel(const Args a, int block_columns) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);         // (sequence, head, column)
  const int64_t per_seq = (int64_t)a.c.nkv * a.columns;
  if (w >= per_seq * a.c.seqs) return;
  const int b = (int)(w / per_seq), rest = (int)(w - b * per_seq), head = rest / a.columns, col = rest % a.columns;
  int tiles0;
  const Schedule sch = schedule_of(a, tiles0);
  const uint32_t n_item = padded(reach_of(a, b).tiles, sch.parts);
  uint32_t before = 0;
  for (int i = lane; i < b; i += 32) before += padded(reach_of(a, i).tiles, sch.parts);
  before = __reduce_add_sync(0xffffffffu, before);
  const uint32_t nth = head * a.blocks + col / block_columns;
  const uint32_t begin = before * a.c.nkv * a.blocks + nth * n_item;
  const uint32_t first = begin / sch.share;
  const int parts = (int)((begin + n_item - 1) / sch.share - first) + 1;
  if (parts == 1) return;
  const int64_t item = (int64_t)b * a.c.nkv * a.blocks + nth;
  const int64_t from = ((int64_t)first + item) * block_columns + col % block_columns;
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
  if (!in && lane == 0) atomicMax(a.err, 2);
  T* to = (T*)a.out + b * a.o_seq + row * a.o_row + (int64_t)(head * a.group + col % a.group) * a.o_head + lane * 8;
  if (lane * 8 < a.c.hd)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      store_from_float(to, std::is_same<T, __half>::value ? FBFP_F16 : FBFP_BF16, i, in ? r[i] * inv : 0.f);
}

// Columns that a block holds: more let one unpacking serve more columns, as far as the accumulators
// leave two CTAs an SM.
int column_tiles(int64_t columns, int groups) {
  if (columns <= 8 || 2 * groups > kAccumulators) return 1;
  if (columns <= 16 || 4 * groups > kAccumulators) return 2;
  return 4;
}

struct Plan {
  int nt, blocks, slots, warps;
  int64_t ctas, segments, list;
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
  const int64_t parts = (tiles + kLeast - 1) / kLeast * items;
  // One CTA of twelve warps an SM where that many hold all parts: a part's tiles at once. (One sequence of 384, 8
  // heads of 256: 10.7 -> 9.0 us.)
  p.warps = p.nt == 1 && parts <= kSms ? 12 : 6;
  p.slots = kSms * 12 / p.warps;
  p.ctas = parts < p.slots ? parts : p.slots;
  p.list = (tiles + kLeast) * items;
  p.joins = parts > items || parts > p.slots;
  p.segments = p.ctas + items;
  return p;
}

template <int NG, int NT, int WARPS, typename T>
int launch(const Args& a, const Maps& m, const Plan& p, cudaStream_t st) {
  auto kernel = kv4_attn_kernel<NG, NT, WARPS, T>;
  static bool set[64];
  int dev = 0;
  FBFP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !set[dev]) {
    FBFP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NG, NT, WARPS>::kSmem));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  FBFP_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(Cfg<NG, NT, WARPS>::kThreads), (size_t)Cfg<NG, NT, WARPS>::kSmem, st, a, m));
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
  if constexpr (4 * NG <= kAccumulators)
    if (p.nt == 4) return launch<NG, 4, 6, T>(a, m, p, st);
  if constexpr (2 * NG <= kAccumulators)
    if (p.nt == 2) return launch<NG, 2, 6, T>(a, m, p, st);
  return p.warps == 12 ? launch<NG, 1, 12, T>(a, m, p, st) : launch<NG, 1, 6, T>(a, m, p, st);
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
  return p.joins ? p.segments * 8 * p.nt * (c.hd + 2) * 4 : 0;
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
  FBFP_CHECK_ARG(std::isfinite(scaling * 1.4426950408889634f), "scaling %g is not finite, or its base-2 form is not", (double)scaling);
  if (((uintptr_t)q | (uintptr_t)out) & 15) return set_error(FBFP_ERR_ALIGN, "q and out must be 16-byte aligned");
  FBFP_CHECK_ARG((int64_t)c.seqs * c.nkv * c.positions < ((int64_t)1 << 31), "the cache has 2^31 rows or more");
  if (window > c.positions + rows) window = 0;              // sees everything
  const Plan p = plan_of(c, rows, heads, window);
  FBFP_CHECK_ARG(p.list < ((int64_t)1 << 31), "too many positions, heads and rows");
  FBFP_CHECK_ARG((int64_t)c.seqs * heads * rows < ((int64_t)1 << 31), "too many rows");
  const int64_t need = p.joins ? p.segments * 8 * p.nt * (c.hd + 2) * 4 : 0;
  FBFP_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                 "the workspace must be %lld bytes, 16-byte aligned", (long long)need);
  const int group = (int)(heads / c.nkv);
  Args a{c, q, out, q_seq, q_row, q_head, o_seq, o_row, o_head, (int)window, (int)rows, (int)heads, group,
         (int)rows * group, p.blocks, pos, err, p.slots, scaling * 1.4426950408889634f, (float*)workspace,
         (float*)workspace + p.segments * 8 * p.nt * c.hd};
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
