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
// bound by memory: every input is read once and every output written once.
#include <cuda_fp8.h>

#include "common.cuh"
#include "pdl.cuh"

namespace fbfp {
namespace {

constexpr int kSeg = 512;            // values a warp takes
constexpr int kLane = 16;            // values a lane takes
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

__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b, const __nv_bfloat16*) {
  a = __uint_as_float(u << 16);
  b = __uint_as_float(u & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b, const __half*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }

// 16 values from p (n of them exist, the others read as zero); vec: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load16(const T* p, int n, bool vec, float (&v)[kLane]) {
  if (vec && n >= kLane) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[h];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2(w[i], v[8 * h + 2 * i], v[8 * h + 2 * i + 1], p);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float4 f = reinterpret_cast<const float4*>(p)[h];
        v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = i < n ? to_float(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store16(T* p, int n, bool vec, const float (&v)[kLane]) {
  if (vec && n >= kLane) {
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < kLane / per; ++h) {
      __align__(16) T o[per];
#pragma unroll
      for (int i = 0; i < per; ++i) from_float(v[per * h + i], o[i]);
      reinterpret_cast<uint4*>(p)[h] = *reinterpret_cast<const uint4*>(o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (i < n) from_float(v[i], p[i]);
  }
}

// One warp: quantise its 512 values (16 per lane, zeros past the row's end) of segment `seg` of
// `row` and store values and scale word. Called by whole warps.
__device__ __forceinline__ void quantise_segment(const float (&v)[kLane], int64_t row, int seg, const RowsOut& o) {
  const int lane = threadIdx.x & 31;
  // maximum of |v| as bits: ordered like the values, with NaN above infinity above all others
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < kLane; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, s));
  // 448 = 1.75 * 2^8: the exponent goes up by one where the mantissa is above 1.75
  int c = (int)((amax + 0x1FFFFFu) >> 23) - 8;
  c = amax >= 0x7F800000u ? 255 : (c < 0 ? 0 : c);
  const float inv = c == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)(254 - c) << 23);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE,
                                                 __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv),
                                                 __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  const int64_t k0 = (int64_t)seg * kSeg + lane * kLane;
  uint8_t* q = o.q + row * o.ldq + k0;
  if (k0 + kLane <= o.k) {
    *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (k0 + i < o.k) q[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
  uint32_t word = (uint32_t)c;
#pragma unroll
  for (int b = 1; b < 4; ++b) word |= (uint32_t)__shfl_sync(0xffffffffu, c, 8 * b) << (8 * b);
  // lane 0 holds block 0's byte; past the row's last block the values are zero and c is 0
  if (lane == 0) o.sc[scale_word(row, seg, o.segs)] = word;
  // the last row also zeroes the tile's rows behind it, so that every scale byte is defined
  if (row == o.m - 1)
    for (int64_t r = o.m + lane; r < ((o.m + 127) & ~(int64_t)127); r += 32) o.sc[scale_word(r, seg, o.segs)] = 0u;
}

// ------------------------------------------------------------------------------- quantise, GeGLU
constexpr int kFlatThreads = 256;

// One warp per (row, segment). GEGLU: the row holds gate | up, `k` values each.
template <typename T, bool GEGLU>
__global__ void __launch_bounds__(kFlatThreads) fp8_rows_kernel(const T* x, int64_t ldx, bool vec, const RowsOut o) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kFlatThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / o.segs;
  if (row >= o.m) return;                              // whole warps
  const int seg = (int)(unit - row * o.segs);
  const int64_t k0 = (int64_t)seg * kSeg + lane * kLane;
  const int n = (int)(o.k - k0 < kLane ? o.k - k0 : kLane);
  const T* p = x + row * ldx + k0;
  float v[kLane];
  load16(p, n, vec, v);
  if constexpr (GEGLU) {
    float u[kLane];
    load16(p + o.k, n, vec, u);
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      // gelu_tanh(g) = g (1 + tanh t) / 2 = g / (1 + exp(-2 t)): no cancellation for g < 0
      const float g = v[i];
      const float t2 = 1.5957691216057308f * (g + 0.044715f * g * g * g);   // 2 sqrt(2 / pi) (..)
      v[i] = g / (1.f + expf(-t2)) * u[i];
    }
  }
  quantise_segment(v, row, seg, o);
}

// ------------------------------------------------------------------------------- RMSNorm
__device__ __forceinline__ float cta_sum(float v, float* red) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

// One CTA per row, its values in registers (NV chunks of 16 per thread; a warp's chunks are 512
// consecutive values). MODE 0: RMSNorm(x; w). MODE 1: h = x + resid first, MODE 2:
// h = RMSNorm(x; w_post) + resid; both store round(h) to resid and normalise the unrounded h.
template <typename T, int NV, int MODE>
__global__ void __launch_bounds__(1024) fp8_rmsnorm_kernel(const T* x, int64_t ldx, const T* w, const T* w_post,
                                                           T* resid, int64_t ldr, float eps, bool vec,
                                                           const RowsOut o) {
  pdl_prologue();
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const float rk = (float)o.k;
  float v[NV][kLane];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k0 = (int64_t)(threadIdx.x + i * blockDim.x) * kLane;
    const int n = (int)(o.k - k0 < kLane ? o.k - k0 : kLane);
    load16(x + row * ldx + k0, n, vec, v[i]);
    if constexpr (MODE == 1) {
      float r[kLane];
      load16((const T*)resid + row * ldr + k0, n, vec, r);
#pragma unroll
      for (int e = 0; e < kLane; ++e) v[i][e] += r[e];
      store16(resid + row * ldr + k0, n, vec, v[i]);
    }
#pragma unroll
    for (int e = 0; e < kLane; ++e) ss += v[i][e] * v[i][e];
  }
  float rs = rsqrtf(cta_sum(ss, red[0]) / rk + eps);
  if constexpr (MODE == 2) {
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t k0 = (int64_t)(threadIdx.x + i * blockDim.x) * kLane;
      const int n = (int)(o.k - k0 < kLane ? o.k - k0 : kLane);
      float wv[kLane], r[kLane];
      load16(w_post + k0, n, vec, wv);
      load16((const T*)resid + row * ldr + k0, n, vec, r);
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        v[i][e] = v[i][e] * rs * (1.f + wv[e]) + r[e];
        ss += v[i][e] * v[i][e];
      }
      store16(resid + row * ldr + k0, n, vec, v[i]);
    }
    rs = rsqrtf(cta_sum(ss, red[1]) / rk + eps);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int chunk = threadIdx.x + i * blockDim.x;
    const int seg = chunk >> 5;
    if (seg >= o.segs) break;                          // whole warps
    const int64_t k0 = (int64_t)chunk * kLane;
    const int n = (int)(o.k - k0 < kLane ? o.k - k0 : kLane);
    float wv[kLane];
    load16(w + k0, n, vec, wv);
#pragma unroll
    for (int e = 0; e < kLane; ++e) v[i][e] = v[i][e] * rs * (1.f + wv[e]);
    quantise_segment(v[i], row, seg, o);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

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

template <typename T, bool GEGLU>
cudaError_t launch_flat(const void* x, int64_t ldx, const RowsOut& o, cudaStream_t st) {
  const bool vec = aligned16(x) && (ldx * sizeof(T)) % 16 == 0 && (!GEGLU || (o.k * sizeof(T)) % 16 == 0);
  const int64_t units = o.m * o.segs, per = kFlatThreads / 32;
  return launch_pdl(fp8_rows_kernel<T, GEGLU>, dim3((unsigned)((units + per - 1) / per)), dim3(kFlatThreads), 0, st,
                    reinterpret_cast<const T*>(x), ldx, vec, o);
}

template <typename T, int NV, int MODE>
cudaError_t launch_norm(const void* x, int64_t ldx, const void* w, const void* w_post, void* resid, int64_t ldr,
                        float eps, const RowsOut& o, cudaStream_t st) {
  const bool vec = aligned16(x) && aligned16(w) && (ldx * sizeof(T)) % 16 == 0 &&
                   (MODE == 0 || (aligned16(resid) && (ldr * sizeof(T)) % 16 == 0)) &&
                   (MODE != 2 || aligned16(w_post));
  const int warps = (o.segs + NV - 1) / NV;
  return launch_pdl(fp8_rmsnorm_kernel<T, NV, MODE>, dim3((unsigned)o.m), dim3(32 * warps), 0, st,
                    reinterpret_cast<const T*>(x), ldx, reinterpret_cast<const T*>(w),
                    reinterpret_cast<const T*>(w_post), reinterpret_cast<T*>(resid), ldr, eps, vec, o);
}

template <typename T, int MODE>
cudaError_t norm_by_size(const void* x, int64_t ldx, const void* w, const void* w_post, void* resid, int64_t ldr,
                         float eps, const RowsOut& o, cudaStream_t st) {
  // up to 16384 values a row fits one chunk per thread
  return o.segs <= 32 ? launch_norm<T, 1, MODE>(x, ldx, w, w_post, resid, ldr, eps, o, st)
                      : launch_norm<T, 2, MODE>(x, ldx, w, w_post, resid, ldr, eps, o, st);
}

template <typename T>
cudaError_t norm_by_mode(const void* x, int64_t ldx, const void* w, const void* w_post, void* resid, int64_t ldr,
                         float eps, const RowsOut& o, cudaStream_t st) {
  return !resid ? norm_by_size<T, 0>(x, ldx, w, w_post, resid, ldr, eps, o, st)
         : w_post ? norm_by_size<T, 2>(x, ldx, w, w_post, resid, ldr, eps, o, st)
                  : norm_by_size<T, 1>(x, ldx, w, w_post, resid, ldr, eps, o, st);
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
  FBFP_CHECK_ARG(ldx >= 0 && (!resid || m == 1 || ldr >= k), "bad row stride (ldx %lld, ldr %lld)", (long long)ldx,
                 (long long)ldr);
  const cudaStream_t st = as_stream(stream);
  FBFP_CUDA_TRY(dtype == FBFP_BF16 ? norm_by_mode<__nv_bfloat16>(x, ldx, w, w_post, resid, ldr, eps, o, st)
                : dtype == FBFP_F16 ? norm_by_mode<__half>(x, ldx, w, w_post, resid, ldr, eps, o, st)
                                    : norm_by_mode<float>(x, ldx, w, w_post, resid, ldr, eps, o, st));
  FBFP_LAUNCH_CHECK("fp8_rmsnorm_kernel");
  return FBFP_OK;
}
