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

// A group's 32 values spread over 4 neighbouring lanes, 8 each: the lane's 8 nibbles and the
// group's scale. All lanes of the warp take part. x / s is rounded exactly: the rest x - n s is a
// multiple of the finer of the two's last places and at most s / 2, so fp32 holds it.
__device__ __forceinline__ void kv4_quantise(const float (&x)[8], uint32_t& word, float& s) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  word = 0x88888888u;
  if (top >= 0x7F800000u) {
    s = __uint_as_float(0x7FC00000u);
    return;
  }
  s = kv4_scale(__uint_as_float(top));
  if (s == 0.f) return;
  const float inv = __fdiv_rn(1.f, s);
  const bool slow = !(s > 1e-37f);                   // 1 / s overflows
  word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float n = rintf(slow ? __fdiv_rn(x[i], s) : x[i] * inv);
    const float rest = fmaf(-n, s, x[i]);
    const float twice = 2.f * fabsf(rest);
    if (twice > s || (twice == s && ((int)n & 1))) n += rest > 0.f ? 1.f : -1.f;
    word |= (uint32_t)((int)n + 8) << (4 * i);
  }
}

// The 8 values of a word of a group with scale s.
__device__ __forceinline__ void kv4_values(uint32_t word, float s, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)((int)((word >> (4 * i)) & 15) - 8) * s;
}

}  // namespace fbfp
