// kv4.cuh — the 4-bit key/value cache: groups of 32 values of a head with one bf16 scale,
// whole numbers n in -7..7 held as n + 8, two to a byte.
#pragma once
#include "common.cuh"

namespace fbfp {

// The cache as the kernels see it (C-ABI checks are in kv4_check).
struct Kv4 {
  uint8_t *kv, *vv;              // values of keys and of values
  uint16_t *ks, *vs;             // scales, bf16 bits
  int seqs, nkv, positions, hd, groups;
  // The place of (sequence, head, position), to be multiplied by groups (scales) or 16 groups (bytes).
  __device__ __forceinline__ int64_t at(int b, int h, int64_t p) const {
    return ((int64_t)b * nkv + h) * positions + p;
  }
};

inline int kv4_check(const fbfp_kv4_cache* c, Kv4& o) {
  FBFP_CHECK_ARG(c && c->k_values && c->k_scales && c->v_values && c->v_scales, "null pointer in the cache");
  FBFP_CHECK_ARG(c->seqs >= 1 && c->seqs <= 65535 && c->kv_heads >= 1 && c->kv_heads <= 65535,
                 "bad cache sizes (%lld sequences, %lld heads)", (long long)c->seqs, (long long)c->kv_heads);
  FBFP_CHECK_ARG(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0,
                 "head_dim %lld is not a multiple of 8 up to 256", (long long)c->head_dim);
  FBFP_CHECK_ARG(c->positions >= 32 && c->positions < (1 << 30) && c->positions % 32 == 0,
                 "positions %lld is not a multiple of 32 below 2^30", (long long)c->positions);
  if (((uintptr_t)c->k_values | (uintptr_t)c->k_scales | (uintptr_t)c->v_values | (uintptr_t)c->v_scales) & 15)
    return set_error(FBFP_ERR_ALIGN, "the cache must be 16-byte aligned");
  o = Kv4{(uint8_t*)c->k_values, (uint8_t*)c->v_values, (uint16_t*)c->k_scales, (uint16_t*)c->v_scales,
          (int)c->seqs, (int)c->kv_heads, (int)c->positions, (int)c->head_dim, (int)((c->head_dim + 31) / 32)};
  return FBFP_OK;
}

// Packed row r: its sequence (-1: nobody's) and its place in it. Any contents of `starts` give a
// sequence below seqs or none.
__device__ __forceinline__ int packed_seq(int64_t r, const int32_t* starts, int seqs, int64_t& place) {
  if (!starts) {
    place = 0;
    return r < seqs ? (int)r : -1;
  }
  int lo = 0, hi = seqs;                 // the last b with starts[b] <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(starts + mid) <= r) lo = mid;
    else hi = mid;
  }
  place = r - __ldg(starts + lo);
  return place >= 0 && r < __ldg(starts + lo + 1) ? lo : -1;
}

// The bf16 nearest to top / 7 (top >= 0, finite): the fp32 quotient rounded again, except that a
// quotient which fp32 rounded onto the middle of two bf16 goes to the side it came from.
__device__ __forceinline__ float kv4_scale(float top) {
  float q = __fdiv_rn(top, 7.f);
  if ((__float_as_uint(q) & 0xFFFFu) == 0x8000u) {
    const float rest = fmaf(-q, 7.f, top);           // exact
    if (rest != 0.f) q = __uint_as_float(__float_as_uint(q) + (rest > 0.f ? 1 : -1));
  }
  return __bfloat162float(__float2bfloat16_rn(q));
}

// A group's 32 values spread over 4 neighbouring lanes, 8 each, `top` the bits of the lane's largest
// magnitude: the lane's 8 nibbles and the group's scale. All lanes of the warp take part.
// WIDE: values of more than 16 bits. A quotient x / s is refined once, y + (x - y s) / s, which leaves it
// exact where fp32 holds it, halves among that. Of values of 16 bits no other quotient comes near a half
// (2 x - (2 n + 1) s is a multiple of both's last places: 2^-13 of s at least), so y rounds as x / s does.
// Wider values decide by the rest x - n s, which fp32 holds: a multiple of the finer of both's last
// places and at most s / 2.
template <bool WIDE>
__device__ __forceinline__ void kv4_quantise(const float (&x)[8], uint32_t top, uint32_t& word, float& s) {
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  word = 0x88888888u;
  if (top >= 0x7F800000u) {
    s = __uint_as_float(0x7FC00000u);
    return;
  }
  s = kv4_scale(__uint_as_float(top));
  if (s == 0.f) return;
  const float up = s < 1e-30f ? 0x1p100f : 1.f;      // where 1 / s could overflow and x - n s be subnormal: exact
  const float t = s * up, inv = __frcp_rn(t);
  // n + 8 comes out in the low bits of 1.5 2^23 + 8, rounded to even; the sum of those words times 16^i is the
  // nibbles' word and what the upper bits add to it
  word = 0u - (uint32_t)(0x4B400000ull * 0x11111111ull);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = x[i] * up;
    float y = z * inv;
    if constexpr (WIDE) {
      y = rintf(y);
      const float rest = fmaf(-y, t, z);
      const float twice = 2.f * fabsf(rest);
      if (twice > t || (twice == t && ((int)y & 1))) y += rest > 0.f ? 1.f : -1.f;
    } else {
      y = fmaf(fmaf(-y, t, z), inv, y);
    }
    if (up != 1.f) y = fminf(fmaxf(y, -7.f), 7.f);   // the lowest subnormal scales may lie far below max|x| / 7
    word += __float_as_uint(y + 12582920.f) << (4 * i);
  }
}
template <bool WIDE>
__device__ __forceinline__ void kv4_quantise(const float (&x)[8], uint32_t& word, float& s) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  kv4_quantise<WIDE>(x, top, word, s);
}

// The 8 values of a word of a group with scale s.
__device__ __forceinline__ void kv4_values(uint32_t word, float s, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)                        // n in the low bits of 2^23, minus 2^23 + 8: exact
    x[i] = (__uint_as_float(0x4B000000u | ((word >> (4 * i)) & 15u)) - 8388616.f) * s;
}

}  // namespace fbfp
