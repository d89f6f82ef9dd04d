// fp8_rows.cu — rows of 8-bit values with a power-of-two scale per 128: quantisation of rows as
// they are, of RMSNorm outputs (with the residual's addition) and of the GeGLU activation. These
// are the operands of the block-scaled product (fp8_gemm.cu).
//
// A block of 128 values x with a = max|x| gets the scale 2^(c - 127), c the smallest integer >= 0
// with a / 2^(c - 127) <= 448 (the largest e4m3 value): the exponent of a / 448 rounded up, read
// off the bits of a. The values x * 2^(127 - c) are exact in fp32, so the one rounding is to e4m3
// (nearest even: at most 2^-4 relative, or 2^-10 of the scale below its normal range). A block
// that holds an infinity or a NaN gets c = 255 (the scale's NaN) and NaN values.
//
// A warp takes 512 consecutive values of a row (4 blocks, one scale word), 16 per lane: a block's
// maximum is a reduction over 8 lanes, and the four scale bytes leave as one 32-bit store into the
// 128-row x 4-block tiles that the tensor core's scale copies take as they are. All of it is
// bound by memory: every input is read once and every output written once. Measured (in a graph
// over more data than L2 holds): quantise 3840 x 15360 fp32 44.4 us (6.65 TB/s), 8192 x 8192 bf16
// 33.5 us (6.0 TB/s); GeGLU 2048 x 15360 bf16 26.7 us (5.9 TB/s), fp32 45.9 us (6.2 TB/s), 2047 x
// 15001, whose rows start anywhere, 35.1 and 47.7 us; residual addition and norm of 8192 x 8192
// bf16 81.5 us (5.8 TB/s); post-norm, addition and norm of 2048 x 3840 bf16 13.2 us (4.2 TB/s: a team
// of warps is in one row at a time and stopped twice in it), 2048 x 3841 25.4 us, one row 2.5 us.
#include <cuda_fp8.h>

#include "common.cuh"
#include "pdl.cuh"
#include "tc_host.h"

namespace fbfp {
namespace {

constexpr int kSeg = 512;            // values a warp takes
constexpr int kLane = 16;            // values a lane takes, as pairs (the fp32 arithmetic is paired)
constexpr int kPairs = kLane / 2;
constexpr int kNormMaxK = 32768;     // the longest row of the norm kernel (1024 threads x 2 chunks)

struct RowsOut {
  uint8_t* q;                        // e4m3 values, row pitch ldq (a multiple of 16)
  int64_t ldq;
  uint32_t* sc;                      // scale tiles
  int64_t m, k;
  int segs;                          // ceil(k / 512): scale words of a row
};

__device__ __forceinline__ int64_t scale_word(int64_t row, int seg, int segs) {
  return ((row >> 7) * segs + seg) * 128 + (row & 31) * 4 + ((row & 127) >> 5);
}

__device__ __forceinline__ float2 unpack2(uint32_t u, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ uint32_t pack2(float2 f, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float2 f, const __half*) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void ld32(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p) : "memory");
}
__device__ __forceinline__ void st32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// The bytes of a tensor, from its first value to its last.
struct Span {
  const char *lo, *hi;
};

// Two kinds of rows. VEC: rows that start on 32 bytes and hold a multiple of 16 values, moved in whole
// 32-byte sectors. Not VEC: any other, moved in the aligned 16-byte vectors that hold them and
// shifted into place (by the same number of bytes in all lanes of a warp). They are separate
// kernels: branches between the two would cost instruction fetches that short rows cannot hide.

// Words out[0..N) = the bytes of in[0..N + 4) from byte s (0..14, even) on.
template <int N>
__device__ __forceinline__ void shift_words(uint32_t (&in)[N + 4], int s, uint32_t (&out)[N]) {
  if (s & 8) {
#pragma unroll
    for (int i = 0; i < N + 2; ++i) in[i] = in[i + 2];
  }
  if (s & 4) {
#pragma unroll
    for (int i = 0; i < N + 1; ++i) in[i] = in[i + 1];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(in[i], in[i + 1], 8 * (s & 2));
}

// A lane's 16 consecutive values of a segment as they lie in memory: loaded early, unpacked where
// they are needed. Not VEC: the vectors that hold them, `shift` the bytes before the first value,
// `mine` how many of the values exist.
template <bool VEC, typename T>
struct Raw16 {
  static constexpr int kWords = kLane * sizeof(T) / 4;
  uint32_t w[kWords + (VEC ? 0 : 4)];
  int shift, mine;
};

// p: the segment's first value; n of the segment's values exist (the others read as zero).
template <bool VEC, typename T>
__device__ __forceinline__ Raw16<VEC, T> load16(const T* p, int n, Span t) {
  Raw16<VEC, T> r;
  constexpr int words = Raw16<VEC, T>::kWords;
  const int lane = threadIdx.x & 31;
  const char* q = reinterpret_cast<const char*>(p + lane * kLane);
  r.mine = n - lane * kLane;
  r.shift = 0;
#pragma unroll
  for (int i = 0; i < words + (VEC ? 0 : 4); ++i) r.w[i] = 0;
  if constexpr (VEC) {
    if (r.mine > 0) {
#pragma unroll
      for (int h = 0; h < words; h += 8) ld32(q + 4 * h, r.w + h);
    }
  } else {
    const int s = (int)((uintptr_t)q & 15);
    const int bytes = s + (r.mine < kLane ? r.mine : kLane) * (int)sizeof(T);   // up to the last existing value
    const char* base = q - s;
    if (r.mine > 0 && base >= t.lo && base + ((bytes + 15) & ~15) <= t.hi) {
      r.shift = s;
#pragma unroll
      for (int h = 0; h < words + 4; h += 4)
        if (4 * h < bytes) {
          const uint4 u = *reinterpret_cast<const uint4*>(base + 4 * h);
          r.w[h] = u.x; r.w[h + 1] = u.y; r.w[h + 2] = u.z; r.w[h + 3] = u.w;
        }
    } else {                                             // a vector would reach past the tensor: value by value
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        if (i < r.mine) {
          if constexpr (sizeof(T) == 4) r.w[i] = reinterpret_cast<const uint32_t*>(q)[i];
          else r.w[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[i] << (16 * (i & 1));
        }
      }
    }
  }
  return r;
}

template <bool VEC, typename T>
__device__ __forceinline__ void unpack16(const Raw16<VEC, T>& r, float2 (&v)[kPairs]) {
  constexpr int words = Raw16<VEC, T>::kWords;
  uint32_t w[words];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < words; ++i) w[i] = r.w[i];
  } else {
    uint32_t in[words + 4];
#pragma unroll
    for (int i = 0; i < words + 4; ++i) in[i] = r.w[i];
    shift_words<words>(in, r.shift, w);
    if (r.mine < kLane) {                                // behind the row's end
#pragma unroll
      for (int i = 0; i < words; ++i) {
        const int left = r.mine * (int)sizeof(T) - 4 * i;
        w[i] &= left >= 4 ? 0xFFFFFFFFu : left > 0 ? 0xFFFFu : 0u;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if constexpr (sizeof(T) == 4)
      v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else
      v[i] = unpack2(w[i], (const T*)nullptr);
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store16(T* p, int n, const float2 (&v)[kPairs]) {
  constexpr int words = kLane * sizeof(T) / 4;
  uint32_t w[words];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(v[i].x);
      w[2 * i + 1] = __float_as_uint(v[i].y);
    } else {
      w[i] = pack2(v[i], (const T*)nullptr);
    }
  }
  const int lane = threadIdx.x & 31;
  T* q = p + lane * kLane;
  if constexpr (VEC) {
    if (lane * kLane < n) {
#pragma unroll
      for (int h = 0; h < words; h += 8) st32(reinterpret_cast<uint32_t*>(q) + h, w + h);
    }
  } else {
    // aligned vectors of this lane's values and the next lane's first, as far as the segment's
    // values fill them; what is left at either end value by value
    constexpr int G = 16 / sizeof(T);                    // values of a vector
    const int s = (int)((uintptr_t)q & 15), lead = s ? (16 - s) / (int)sizeof(T) : 0;
    const int end = n >= lead ? lead + (n - lead) / G * G : 0, v0 = lane * kLane;
    uint32_t in[words + 4], out[words];
#pragma unroll
    for (int i = 0; i < words; ++i) in[i] = w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) in[words + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
    shift_words<words>(in, (16 - s) & 15, out);
#pragma unroll
    for (int h = 0; h < kLane / G; ++h)
      if (v0 + lead + (h + 1) * G <= end)
        reinterpret_cast<uint4*>(q + lead)[h] = make_uint4(out[4 * h], out[4 * h + 1], out[4 * h + 2], out[4 * h + 3]);
    if (v0 < lead || v0 + kLane > end) {
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        if ((v0 + i < lead || v0 + i >= end) && v0 + i < n) {
          if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(q)[i] = w[i];
          else reinterpret_cast<uint16_t*>(q)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    }
  }
}

// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float amax3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Scale byte of a block whose values' magnitude bits have the maximum amax, and the factor
// 2^(127 - c). 448 = 1.75 * 2^8: the exponent goes up by one where the mantissa is above 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int c = (int)((amax + 0x1FFFFFu) >> 23) - 8;
  return amax >= 0x7F800000u ? 255 : (c < 0 ? 0 : c);
}
__device__ __forceinline__ float scale_inverse(int c) {
  return c == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)(254 - c) << 23);
}

// One warp: quantise its 512 values (zeros past the row's end) of segment `seg` of `row` and store
// values and scale word. Called by whole warps. Across lanes the maximum of |v| is taken on its
// bits, which are ordered like the values, with NaN above infinity above all others.
template <bool VEC>
__device__ __forceinline__ void quantise_segment(const float2 (&v)[kPairs], int64_t row, int seg, const RowsOut& o) {
  const int lane = threadIdx.x & 31;
  uint8_t* q = o.q + row * o.ldq + (int64_t)seg * kSeg + lane * kLane;
  const int64_t left = o.k - (int64_t)seg * kSeg - lane * kLane;
  const int mine = left < kLane ? (int)left : kLane;     // of this lane's values exist
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) top = amax3(top, v[i].x, v[i].y);
  uint32_t amax = __float_as_uint(top);
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, s));
  const int c = scale_byte(amax);
  const float2 inv = make_float2(scale_inverse(c), scale_inverse(c));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(__fmul2_rn(v[2 * i], inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(__fmul2_rn(v[2 * i + 1], inv), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  if (VEC ? mine > 0 : mine >= kLane) {
    *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (!VEC) {
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (i < mine) q[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
  uint32_t word = (uint32_t)c;
#pragma unroll
  for (int b = 1; b < 4; ++b) word |= (uint32_t)__shfl_sync(0xffffffffu, c, 8 * b) << (8 * b);
  // lane 0's word is right; past the row's last block the values are zero and so are the bytes
  if (lane == 0) o.sc[scale_word(row, seg, o.segs)] = word;
  // the last row also zeroes the tile's rows behind it, so that every scale byte is defined
  if (row == o.m - 1)
    for (int64_t r = o.m + lane; r < ((o.m + 127) & ~(int64_t)127); r += 32) o.sc[scale_word(r, seg, o.segs)] = 0u;
}

__device__ __forceinline__ int left_of(int64_t k, int seg) {   // values of the row from segment `seg` on
  const int64_t n = k - (int64_t)seg * kSeg;
  return n > kSeg ? kSeg : (int)n;                             // 0 or less: none
}

// ------------------------------------------------------------------------------- quantise, GeGLU
constexpr int kFlatThreads = 256;

// gelu_tanh(g) = g (1 + tanh t) / 2 = g / (1 + exp(-2 t)), t = sqrt(2 / pi) (g + 0.044715 g^3): no
// cancellation for negative g. The exponent e is taken to base 2, log2(e) in its constants.
// EXACT, for fp32 inputs: with s = 2^-|e|, g (s or 1) / (1 + s), whose denominator lies in [1, 2]
// for every gate and whose reciprocal's quotient is corrected from its residual. Else g / (1 + 2^e)
// as it is. Either way a very negative gate (a mask of the lowest value, say) gives 0: s flushes to
// 0 below 2^-126, as does the reciprocal of a denominator above 2^126, off by at most 10.1 * 2^-126
// (gates between -10.0 and -10.3). (16-bit inputs round to the same 8-bit values without the
// correction, in every case compared with fp64 and with the divided form; it costs them 7%.)
template <bool EXACT>
__device__ __forceinline__ float2 gelu_tanh(float2 g) {
  const float c1 = 2.302208198144325f, c2 = 0.1029432395800235f;   // 2 log2(e) sqrt(2 / pi) (1, 0.044715)
  const float2 t = __fmul2_rn(g, __ffma2_rn(make_float2(-c2, -c2), __fmul2_rn(g, g), make_float2(-c1, -c1)));
  float2 e, r;
  if constexpr (EXACT) {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(-fabsf(t.x)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(-fabsf(t.y)));
    const float2 n = __fmul2_rn(g, make_float2(t.x > 0.f ? e.x : 1.f, t.y > 0.f ? e.y : 1.f));
    e = __fadd2_rn(e, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    const float2 q = __fmul2_rn(n, r);
    return __ffma2_rn(__ffma2_rn(make_float2(-q.x, -q.y), e, n), r, q);
  } else {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = __fadd2_rn(e, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return __fmul2_rn(g, r);
  }
}

// One warp per (row, segment). GEGLU: the row holds gate | up, `k` values each.
template <typename T, bool GEGLU, bool VEC>
__global__ void __launch_bounds__(kFlatThreads) fp8_rows_kernel(const T* x, int64_t ldx, const Span t, const RowsOut o) {
  pdl_prologue();
  const int64_t unit = (int64_t)blockIdx.x * (kFlatThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / o.segs;
  if (row >= o.m) return;                              // whole warps
  const int seg = (int)(unit - row * o.segs), n = left_of(o.k, seg);
  const T* p = x + row * ldx + (int64_t)seg * kSeg;
  float2 v[kPairs];
  if constexpr (GEGLU) {
    const Raw16<VEC, T> gr = load16<VEC>(p, n, t), ur = load16<VEC>(p + o.k, n, t);
    float2 u[kPairs];
    unpack16(gr, v);
    unpack16(ur, u);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) v[i] = __fmul2_rn(gelu_tanh<sizeof(T) == 4>(v[i]), u[i]);
  } else {
    unpack16(load16<VEC>(p, n, t), v);
  }
  quantise_segment<VEC>(v, row, seg, o);
}

// ------------------------------------------------------------------------------- RMSNorm
// A team of warps takes a row, a warp NV segments of it, in registers; a CTA has one team or
// several and goes on to further rows, whose values are on their way while a row is worked on
// (kEarly: all but rows above 16384 values, whose 1024 threads have 64 registers each, and long
// fp32 rows). The weights come from L1. MODE 0: RMSNorm(x; w). MODE 1: h = x + resid first,
// MODE 2: h = RMSNorm(x; w_post) + resid; both store round(h) to resid and normalise the
// unrounded h.
struct NormArgs {
  int64_t ldx, ldr;
  float eps, inv_k;
  Span xs, rs, ws, ps;                                   // of x, resid, w, w_post
  int team;                                              // warps per row
};

// 1 / sqrt(ss / k + eps). A relative error here moves a whole row, and with it the share of its
// values that round to the other side in 8 bits: so the quotient (a product with inv_k = 1 / k) and
// the approximate root (2 units in the last place) each get a correction from their residual.
__device__ __forceinline__ float row_scale(float ss, float k, float inv_k, float eps) {
  float q = ss * inv_k;
  q = q < 3.4e38f ? fmaf(fmaf(-q, k, ss), inv_k, q) : q;
  const float a = q + eps, y = rsqrtf(a);
  return y > 0.f && a > 0.f ? fmaf(0.5f * y, fmaf(-a * y, y, 1.f), y) : y;   // not for a = 0 or infinity
}

__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Sum over the warps of a team; red: MAXW floats of the team, zero where it has fewer warps.
template <int MAXW>
__device__ __forceinline__ float team_sum(float2 p, float* red, int warp) {
  float v = p.x + p.y;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  float2 t = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < MAXW; w += 4) {
    const float4 q = *reinterpret_cast<const float4*>(red + w);
    t = __fadd2_rn(t, __fadd2_rn(make_float2(q.x, q.y), make_float2(q.z, q.w)));
  }
  return t.x + t.y;
}

template <typename T, int NV, int MODE, int THREADS, int MINB, bool VEC>
__global__ void __launch_bounds__(THREADS, MINB) fp8_rmsnorm_kernel(const T* x, const T* w, const T* w_post, T* resid,
                                                                    const NormArgs a, const RowsOut o) {
  pdl_prologue();
  constexpr bool kEarly = THREADS < 1024 && (NV == 1 || sizeof(T) == 2);
  constexpr int kWarps = THREADS / 32, kTeams = THREADS <= 256 ? kWarps : 1;   // at most, a CTA
  __shared__ __align__(16) float reds[2][kTeams * kWarps];
  for (int i = threadIdx.x; i < 2 * kTeams * kWarps; i += blockDim.x) (&reds[0][0])[i] = 0.f;
  __syncthreads();
  const int warp = threadIdx.x >> 5, teams = (int)(blockDim.x >> 5) / a.team;
  const int seg0 = warp % a.team;                        // this warp's segments: seg0 + i * team
  float* red = reds[0] + warp / a.team * kWarps;         // this team's sums, two rooms in turn
  const int64_t step = (int64_t)gridDim.x * teams;
  int64_t row = (int64_t)blockIdx.x * teams + warp / a.team;
  const float rk = (float)o.k;
  const T *xp = x + row * a.ldx, *rp = resid + row * a.ldr;
  Raw16<VEC, T> xr[NV], rr[NV];
  if constexpr (kEarly) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int seg = seg0 + i * a.team, n = row < o.m ? left_of(o.k, seg) : 0;
      xr[i] = load16<VEC>(xp + seg * kSeg, n, a.xs);
      if constexpr (MODE > 0) rr[i] = load16<VEC>(rp + seg * kSeg, n, a.rs);
    }
  }
  int turn = 0;
#pragma unroll 1
  for (int64_t base = (int64_t)blockIdx.x * teams; base < o.m; base += step, row += step) {
    const bool live = row < o.m, more = row + step < o.m;   // a team past the last row takes part in the sums only
    T* const now = resid + row * a.ldr;                      // this row of the residual
    float2 v[NV][kPairs];
    float2 ss = make_float2(0.f, 0.f);
    if constexpr (kEarly) xp += step * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int seg = seg0 + i * a.team, all = left_of(o.k, seg), n = live ? all : 0;
      if constexpr (!kEarly) xr[i] = load16<VEC>(x + row * a.ldx + seg * kSeg, n, a.xs);
      unpack16(xr[i], v[i]);
      if constexpr (kEarly) xr[i] = load16<VEC>(xp + seg * kSeg, more ? all : 0, a.xs);
      if constexpr (MODE == 1) {
        if constexpr (!kEarly) rr[i] = load16<VEC>((const T*)now + seg * kSeg, n, a.rs);
        float2 r[kPairs];
        unpack16(rr[i], r);
        if constexpr (kEarly) rr[i] = load16<VEC>((const T*)now + step * a.ldr + seg * kSeg, more ? all : 0, a.rs);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) v[i][e] = __fadd2_rn(v[i][e], r[e]);
        store16<VEC>(now + seg * kSeg, n, v[i]);
      }
#pragma unroll
      for (int e = 0; e < kPairs; ++e) ss = __ffma2_rn(v[i][e], v[i][e], ss);
    }
    float rs = row_scale(team_sum<kWarps>(ss, red + turn, seg0), rk, a.inv_k, a.eps);
    turn ^= kTeams * kWarps;
    if constexpr (MODE == 2) {
      ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int seg = seg0 + i * a.team, all = left_of(o.k, seg), n = live ? all : 0;
        if constexpr (!kEarly) rr[i] = load16<VEC>((const T*)now + seg * kSeg, n, a.rs);
        float2 wv[kPairs];
        unpack16(load16<VEC>(w_post + seg * kSeg, n, a.ps), wv);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {               // y = v rs, y + y w
          v[i][e] = __fmul2_rn(v[i][e], both(rs));
          v[i][e] = __ffma2_rn(v[i][e], wv[e], v[i][e]);
        }
        unpack16(rr[i], wv);
        if constexpr (kEarly) rr[i] = load16<VEC>((const T*)now + step * a.ldr + seg * kSeg, more ? all : 0, a.rs);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          v[i][e] = __fadd2_rn(v[i][e], wv[e]);
          ss = __ffma2_rn(v[i][e], v[i][e], ss);
        }
        store16<VEC>(now + seg * kSeg, n, v[i]);
      }
      rs = row_scale(team_sum<kWarps>(ss, red + turn, seg0), rk, a.inv_k, a.eps);
      turn ^= kTeams * kWarps;
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int seg = seg0 + i * a.team;
        if (seg >= o.segs) break;                        // whole warps
        float2 wv[kPairs];
        unpack16(load16<VEC>(w + seg * kSeg, left_of(o.k, seg), a.ws), wv);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          v[i][e] = __fmul2_rn(v[i][e], both(rs));
          v[i][e] = __ffma2_rn(v[i][e], wv[e], v[i][e]);
        }
        quantise_segment<VEC>(v[i], row, seg, o);
      }
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Whether rows whose addresses and byte strides (or'ed) are these start on 32 bytes and hold whole
// lanes' values.
bool whole_sectors(uint64_t bits, int64_t k) { return (bits & 31) == 0 && k % kLane == 0; }
uint64_t bits_of(const void* p) { return (uint64_t)(uintptr_t)p; }

// Arguments common to the three entries; fills o.
int rows_out(int64_t m, int64_t k, void* values, int64_t ldv, void* scales, RowsOut& o) {
  FBFP_CHECK_ARG(values && scales, "null pointer");
  FBFP_CHECK_ARG(m >= 1 && m < ((int64_t)1 << 31) && k >= 1 && k < ((int64_t)1 << 31), "bad sizes (m %lld, k %lld)",
                 (long long)m, (long long)k);
  FBFP_CHECK_ARG(ldv >= k && ldv % 16 == 0 && aligned16(values),
                 "values must be 16-byte aligned with rows a multiple of 16 apart (ldv %lld)", (long long)ldv);
  FBFP_CHECK_ARG(aligned16(scales), "scales must be 16-byte aligned");
  o.q = reinterpret_cast<uint8_t*>(values);
  o.ldq = ldv;
  o.sc = reinterpret_cast<uint32_t*>(scales);
  o.m = m;
  o.k = k;
  o.segs = (int)((k + kSeg - 1) / kSeg);
  return FBFP_OK;
}

template <typename T>
Span span(const void* p, int64_t rows, int64_t ld, int64_t len) {
  const char* c = reinterpret_cast<const char*>(p);
  return Span{c, c ? c + ((rows - 1) * ld + len) * (int64_t)sizeof(T) : c};
}

template <typename T, bool GEGLU>
cudaError_t launch_flat(const void* x, int64_t ldx, const RowsOut& o, cudaStream_t st) {
  const bool vec = whole_sectors(bits_of(x) | (uint64_t)ldx * sizeof(T), o.k);
  const int64_t units = o.m * o.segs, per = kFlatThreads / 32;
  return launch_pdl(vec ? fp8_rows_kernel<T, GEGLU, true> : fp8_rows_kernel<T, GEGLU, false>,
                    dim3((unsigned)((units + per - 1) / per)), dim3(kFlatThreads), 0, st,
                    reinterpret_cast<const T*>(x), ldx, span<T>(x, o.m, ldx, GEGLU ? 2 * o.k : o.k), o);
}

struct NormPtrs {
  const void *x, *w, *w_post;
  void* resid;
};

template <typename T, int NV, int MODE, int THREADS, int MINB, bool VEC>
cudaError_t launch_norm(const NormPtrs& p, NormArgs a, const RowsOut& o, int nsm, cudaStream_t st) {
  a.team = (o.segs + NV - 1) / NV;
  a.xs = span<T>(p.x, o.m, a.ldx, o.k);
  a.rs = span<T>(p.resid, o.m, a.ldr, o.k);
  a.ws = span<T>(p.w, 1, 0, o.k);
  a.ps = span<T>(p.w_post, 1, 0, o.k);
  const int teams = THREADS <= 256 ? THREADS / 32 / a.team : 1;   // rows of a CTA at a time
  const int64_t want = (o.m + teams - 1) / teams;
  const int64_t room = (int64_t)nsm * MINB;
  return launch_pdl(fp8_rmsnorm_kernel<T, NV, MODE, THREADS, MINB, VEC>, dim3((unsigned)(want < room ? want : room)),
                    dim3(32 * a.team * teams), 0, st, reinterpret_cast<const T*>(p.x),
                    reinterpret_cast<const T*>(p.w), reinterpret_cast<const T*>(p.w_post),
                    reinterpret_cast<T*>(p.resid), a, o);
}

template <typename T, int MODE>
cudaError_t norm_by_size(const NormPtrs& p, NormArgs a, const RowsOut& o, int nsm, cudaStream_t st) {
  const bool vec = whole_sectors(bits_of(p.x) | bits_of(p.w) | bits_of(p.resid) | bits_of(p.w_post) |
                                     (uint64_t)a.ldx * sizeof(T) | (MODE ? (uint64_t)a.ldr * sizeof(T) : 0),
                                 o.k);
  // CTAs per SM by the registers of a row's 16 values a thread (twice as many words in fp32)
  constexpr int kThree = sizeof(T) == 2 ? 3 : 2, kTwo = sizeof(T) == 2 ? 2 : 1;
  if (!vec)
    return o.segs <= 8    ? launch_norm<T, 1, MODE, 256, 2, false>(p, a, o, nsm, st)
           : o.segs <= 16 ? launch_norm<T, 1, MODE, 512, 1, false>(p, a, o, nsm, st)
           : o.segs <= 32 ? launch_norm<T, 2, MODE, 512, 1, false>(p, a, o, nsm, st)
                          : launch_norm<T, 2, MODE, 1024, 1, false>(p, a, o, nsm, st);
  return o.segs <= 8    ? launch_norm<T, 1, MODE, 256, kThree, true>(p, a, o, nsm, st)
         : o.segs <= 16 ? launch_norm<T, 1, MODE, 512, kTwo, true>(p, a, o, nsm, st)
         : o.segs <= 32 ? launch_norm<T, 2, MODE, 512, 1, true>(p, a, o, nsm, st)
                        : launch_norm<T, 2, MODE, 1024, 1, true>(p, a, o, nsm, st);
}

template <typename T>
cudaError_t norm_by_mode(const NormPtrs& p, const NormArgs& a, const RowsOut& o, int nsm, cudaStream_t st) {
  return !p.resid ? norm_by_size<T, 0>(p, a, o, nsm, st)
         : p.w_post ? norm_by_size<T, 2>(p, a, o, nsm, st)
                    : norm_by_size<T, 1>(p, a, o, nsm, st);
}

template <bool GEGLU>
int flat_entry(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, void* values, int64_t ldv, void* scales,
               void* stream) {
  FBFP_CHECK_ARG(x, "null pointer");
  FBFP_CHECK_ARG(dtype_ok(dtype), "bad dtype %d", dtype);
  RowsOut o;
  const int rc = rows_out(m, k, values, ldv, scales, o);
  if (rc != FBFP_OK) return rc;
  FBFP_CHECK_ARG(ldx >= 0, "bad row stride %lld", (long long)ldx);   // 0: one row for all
  FBFP_CHECK_ARG((uintptr_t)x % dtype_size(dtype) == 0, "values must be aligned to their type");
  FBFP_CHECK_ARG(m * o.segs < ((int64_t)1 << 33), "too many values (m %lld, k %lld)", (long long)m, (long long)k);
  const cudaStream_t st = as_stream(stream);
  const cudaError_t e = dtype == FBFP_BF16 ? launch_flat<__nv_bfloat16, GEGLU>(x, ldx, o, st)
                        : dtype == FBFP_F16 ? launch_flat<__half, GEGLU>(x, ldx, o, st)
                                            : launch_flat<float, GEGLU>(x, ldx, o, st);
  FBFP_CUDA_TRY(e);
  FBFP_LAUNCH_CHECK("fp8_rows_kernel");
  return FBFP_OK;
}

}  // namespace
}  // namespace fbfp

using namespace fbfp;

extern "C" int64_t fbfp_fp8_scale_bytes(int64_t rows, int64_t k) {
  if (rows < 1 || k < 1) return -1;
  return (rows + 127) / 128 * ((k + kSeg - 1) / kSeg) * 512;
}

extern "C" int fbfp_fp8_quantize(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, void* values,
                                 int64_t ldv, void* scales, void* stream) {
  return flat_entry<false>(x, x_dtype, m, k, ldx, values, ldv, scales, stream);
}

extern "C" int fbfp_fp8_geglu(const void* gate_up, int dtype, int64_t m, int64_t inter, int64_t ldx, void* values,
                              int64_t ldv, void* scales, void* stream) {
  return flat_entry<true>(gate_up, dtype, m, inter, ldx, values, ldv, scales, stream);
}

extern "C" int fbfp_fp8_rmsnorm(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, const void* w,
                                const void* w_post, void* resid, int64_t ldr, float eps, void* values, int64_t ldv,
                                void* scales, void* stream) {
  FBFP_CHECK_ARG(x && w, "null pointer");
  FBFP_CHECK_ARG(dtype_ok(dtype), "bad dtype %d", dtype);
  FBFP_CHECK_ARG(!w_post || resid, "a post-norm weight needs the residual it is added to");
  RowsOut o;
  const int rc = rows_out(m, k, values, ldv, scales, o);
  if (rc != FBFP_OK) return rc;
  FBFP_CHECK_ARG(k <= kNormMaxK, "rows of at most %d values (got %lld)", kNormMaxK, (long long)k);
  FBFP_CHECK_ARG(((uintptr_t)x | (uintptr_t)w | (uintptr_t)w_post | (uintptr_t)resid) % dtype_size(dtype) == 0,
                 "values must be aligned to their type");
  FBFP_CHECK_ARG(ldx >= 0 && (!resid || m == 1 || ldr >= k), "bad row stride (ldx %lld, ldr %lld)", (long long)ldx,
                 (long long)ldr);
  int dev = 0;
  FBFP_CUDA_TRY(cudaGetDevice(&dev));
  const NormPtrs p{x, w, w_post, resid};
  const NormArgs a{ldx, ldr, eps, 1.f / (float)k, {}, {}, {}, {}, 0};
  const int nsm = sm_count(dev);
  const cudaStream_t st = as_stream(stream);
  FBFP_CUDA_TRY(dtype == FBFP_BF16  ? norm_by_mode<__nv_bfloat16>(p, a, o, nsm, st)
                : dtype == FBFP_F16 ? norm_by_mode<__half>(p, a, o, nsm, st)
                                    : norm_by_mode<float>(p, a, o, nsm, st));
  FBFP_LAUNCH_CHECK("fp8_rmsnorm_kernel");
  return FBFP_OK;
}
