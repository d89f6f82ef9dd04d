// kv4.cu — writing rows of keys and values into the 4-bit cache, reading ranges of it back, and
// the decoder's append (q/k RMSNorm, rotary embedding and write in one launch).
#include "kv4.cuh"
#include "pdl.cuh"

namespace fbfp {
namespace {

constexpr int kThreads = 256;

struct RowsArg {                 // plain rows of k and v
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head, rows;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// Eight values at p; VEC: p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (VEC) {
    union { uint4 u[sizeof(T) / 2]; T t[8]; } b;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) b.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(b.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(p[i]);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (VEC) {
    union { uint4 u[sizeof(T) / 2]; T t[8]; } b;
#pragma unroll
    for (int i = 0; i < 8; ++i) b.t[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = b.u[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(x[i]);
  }
}

// A row's keys and values are 2 kv_heads heads of pieces of 8 values. So many threads take a row, whole warps, a
// piece each; a CTA takes as many rows as it has threads for, or a part (blockIdx.y) of one row's pieces.
struct Shape {
  int per_row;                   // threads of a row in a CTA
  int rows;                      // rows of a CTA
  int parts;                     // CTAs of a row
};
Shape shape_of(int pieces) {
  const int t = (pieces + 31) / 32 * 32;
  return t < kThreads ? Shape{t, kThreads / t, 1} : Shape{kThreads, 1, (t + kThreads - 1) / kThreads};
}
struct Place {
  int b;                         // sequence, -1: none
  int64_t at;                    // position
};
// Row r's place; a position outside the cache is recorded (by one thread of the row).
__device__ __forceinline__ Place place_of(int64_t r, const Kv4& c, int64_t rows, const int32_t* base, const int32_t* starts,
                                          int32_t* err, bool tell) {
  Place p{-1, 0};
  if (r >= rows) return p;
  p.b = packed_seq(r, starts, c.seqs, p.at);
  if (p.b < 0) return p;
  p.at += __ldg(base + p.b);
  if (p.at < 0 || p.at >= c.positions) {
    if (tell) atomicMax(err, 2);
    p.b = -1;
  }
  return p;
}

// A piece as it is in memory, its largest magnitude's bits (as fp32), and its values.
template <typename T>
struct Raw {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
      T* t = reinterpret_cast<T*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = p[i];
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      const float* f = reinterpret_cast<const float*>(u);
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
      return m;
    } else {                                            // magnitudes in halves order as their bits do
      uint32_t m = __vmaxu2(__vmaxu2(u[0].x & 0x7FFF7FFFu, u[0].y & 0x7FFF7FFFu),
                            __vmaxu2(u[0].z & 0x7FFF7FFFu, u[0].w & 0x7FFF7FFFu));
      m = max(m & 0xFFFFu, m >> 16);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
      else return __float_as_uint(__half2float(__ushort_as_half((uint16_t)m))) & 0x7FFFFFFFu;
    }
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    const T* t = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(t[i]);
  }
};

// Bound by memory: a row's values in, 4.5 bits of each out. A thread takes the same piece of R rows, so that as
// many loads are on their way at once.
template <typename T, bool VEC, int NG, int R>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(Kv4 c, RowsArg r, Shape sh, const int32_t* pos,
                                                             const int32_t* starts, int32_t* err) {
  pdl_prologue();
  constexpr int per_head = 4 * NG;
  if (threadIdx.x / sh.per_row >= sh.rows) return;     // whole warps
  const int64_t row0 = ((int64_t)blockIdx.x * sh.rows + threadIdx.x / sh.per_row) * R;
  const int i = blockIdx.y * sh.per_row + threadIdx.x % sh.per_row;
  const int pieces = 2 * c.nkv * per_head;
  const int h = i / per_head, piece = i % per_head;
  const bool which = h >= c.nkv;
  const int head = which ? h - c.nkv : h;
  const int64_t step = which ? r.v_row : r.k_row;
  const T* from = (which ? (const T*)r.v + head * r.v_head : (const T*)r.k + head * r.k_head) + row0 * step + piece * 8;
  Raw<T> raw[R];                                       // whatever sequence they belong to: the loads need not wait for that
#pragma unroll
  for (int k = 0; k < R; ++k) {
    if (i < pieces && piece * 8 < c.hd && row0 + k < r.rows) raw[k].template load<VEC>(from + k * step);
    else raw[k].zero();
  }
  const auto put = [&](const Raw<T>& x, int64_t to) {
    float v[8];
    uint32_t word;
    float s;
    x.values(v);
    kv4_quantise<sizeof(T) == 4>(v, x.top(), word, s);
    if (to < 0) return;
    reinterpret_cast<uint32_t*>((which ? c.vv : c.kv) + to * 16)[piece] = word;
    if ((piece & 3) == 0) (which ? c.vs : c.ks)[to + (piece >> 2)] = (uint16_t)(__float_as_uint(s) >> 16);
  };
  Place a = place_of(row0, c, r.rows, pos, starts, err, i == 0);
  const Place z = R > 1 ? place_of(row0 + R - 1, c, r.rows, pos, starts, err, i == 0) : a;
  const bool run = R == 1 || (a.b >= 0 && a.b == z.b && z.at - a.at == R - 1);      // rows that follow each other
  const int64_t first = a.b >= 0 && i < pieces ? c.at(a.b, head, a.at) * NG : -1;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    int64_t to = first < 0 ? -1 : first + k * NG;
    if (k > 0 && !run) {
      const Place p = place_of(row0 + k, c, r.rows, pos, starts, err, i == 0);
      to = p.b >= 0 && i < pieces ? c.at(p.b, head, p.at) * NG : -1;
    }
    put(raw[k], to);
  }
}

// Eight values n s of a word as they are stored. bf16: n in bf16 times s, rounded once, as in fp32.
template <typename T, bool VEC>
__device__ __forceinline__ void store_values(T* to, uint32_t word, uint16_t scale) {
  if constexpr (VEC && std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t s2 = scale | (uint32_t)scale << 16;
    uint32_t x[4];                                      // nibbles (i, i + 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = ((word >> (4 * i)) & 0x000F000Fu) | 0x43004300u, off = 0x43084308u;   // 128 + n, less 136
      const __nv_bfloat162 n = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m), *reinterpret_cast<const __nv_bfloat162*>(&off));
      const __nv_bfloat162 v = __hmul2_rn(n, *reinterpret_cast<const __nv_bfloat162*>(&s2));
      x[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410),
                                               __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
  } else {
    float x[8];
    kv4_values(word, bf16_bits_to_float(scale), x);
    store8<T, VEC>(to, x);
  }
}

template <typename T, bool VEC, int NG, int R>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4 c, RowsArg r, Shape sh, const int32_t* first,
                                                            const int32_t* starts, int32_t* err) {
  pdl_prologue();
  constexpr int per_head = 4 * NG;                     // (a last group of fewer than 32 values: some idle)
  if (threadIdx.x / sh.per_row >= sh.rows) return;
  const int64_t row0 = ((int64_t)blockIdx.x * sh.rows + threadIdx.x / sh.per_row) * R;
  const int i = blockIdx.y * sh.per_row + threadIdx.x % sh.per_row;
  const int h = i / per_head, piece = i % per_head;
  if (i >= 2 * c.nkv * per_head || piece * 8 >= c.hd) return;
  const bool which = h >= c.nkv;
  const int head = which ? h - c.nkv : h;
  const int64_t step = which ? r.v_row : r.k_row;
  T* const to = (which ? (T*)r.v + head * r.v_head : (T*)r.k + head * r.k_head) + row0 * step + piece * 8;
  const uint32_t* const values = reinterpret_cast<const uint32_t*>(which ? c.vv : c.kv) + piece;
  const uint16_t* const scales = (which ? c.vs : c.ks) + (piece >> 2);
  const Place a = place_of(row0, c, r.rows, first, starts, err, i == 0);
  const Place z = R > 1 ? place_of(row0 + R - 1, c, r.rows, first, starts, err, i == 0) : a;
  if (R == 1 || (a.b >= 0 && a.b == z.b && z.at - a.at == R - 1)) {     // rows that follow each other
    if (a.b < 0) return;
    const int64_t from = c.at(a.b, head, a.at) * NG;
    uint32_t word[R];
    uint16_t s[R];
#pragma unroll
    for (int k = 0; k < R; ++k) word[k] = __ldg(values + (from + k * NG) * 4), s[k] = __ldg(scales + from + k * NG);
#pragma unroll
    for (int k = 0; k < R; ++k) store_values<T, VEC>(to + k * step, word[k], s[k]);
    return;
  }
  if constexpr (R > 1) {
#pragma unroll 1
    for (int k = 0; k < R; ++k) {
      const Place p = place_of(row0 + k, c, r.rows, first, starts, err, i == 0);
      if (p.b < 0) continue;
      const int64_t from = c.at(p.b, head, p.at) * NG;
      store_values<T, VEC>(to + k * step, __ldg(values + from * 4), __ldg(scales + from));
    }
  }
}

__device__ __forceinline__ float rb(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// One warp per head of a fused q|k|v row, lane l owning values 8 l .. 8 l + 7 (zeros past the head):
// RMSNorm of q and k as a warp sum, the rotation's partner hd / 16 lanes away, then q to its rows
// and k and v to the cache. Rounded to bf16 where the separate norm and rotation round.
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Kv4 c, const __nv_bfloat16* qkv, int64_t rows, int nh,
                                                              const __nv_bfloat16* qnw, const __nv_bfloat16* knw,
                                                              float eps, const __nv_bfloat16* cos_t,
                                                              const __nv_bfloat16* sin_t, const int32_t* pos,
                                                              const int32_t* starts, __nv_bfloat16* q_out,
                                                              int32_t* err) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int all = nh + 2 * c.nkv;
  const int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = w / all;
  const int head = (int)(w - row * all);
  if (row >= rows) return;
  int64_t at;
  const int b = packed_seq(row, starts, c.seqs, at);
  if (b < 0) return;
  at += pos[b];
  if (at < 0 || at >= c.positions) {
    if (lane == 0) atomicMax(err, 2);
    return;
  }
  const bool act = lane * 8 < c.hd;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (act) load8<__nv_bfloat16, true>(qkv + (row * all + head) * c.hd + lane * 8, x);
  if (head < nh + c.nkv) {
    float wv[8], cv[8], sv[8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i], wv[i] = cv[i] = sv[i] = 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float rms = rsqrtf(ss / (float)c.hd + eps);
    if (act) {
      load8<__nv_bfloat16, true>((head < nh ? qnw : knw) + lane * 8, wv);
      load8<__nv_bfloat16, true>(cos_t + at * c.hd + lane * 8, cv);
      load8<__nv_bfloat16, true>(sin_t + at * c.hd + lane * 8, sv);
    }
    const int hl = c.hd >> 4;                         // lanes per half of the head
    const bool low = lane < hl;
    const int partner = (low ? lane + hl : lane - hl) & 31;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = rb(x[i] * rms * (1.f + wv[i]));
#pragma unroll
    for (int i = 0; i < 8; ++i) wv[i] = __shfl_sync(0xffffffffu, x[i], partner);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = act ? rb(rb(x[i] * cv[i]) + rb((low ? -wv[i] : wv[i]) * sv[i])) : 0.f;
  }
  if (head < nh) {
    if (act) store8<__nv_bfloat16, true>(q_out + (row * nh + head) * c.hd + lane * 8, x);
    return;
  }
  uint32_t word;
  float s;
  kv4_quantise<false>(x, word, s);
  if (lane >= 4 * c.groups) return;
  const int which = head >= nh + c.nkv;
  const int64_t to = c.at(b, head - nh - (which ? c.nkv : 0), at) * c.groups;
  reinterpret_cast<uint32_t*>((which ? c.vv : c.kv) + to * 16)[lane] = word;
  if ((lane & 3) == 0) (which ? c.vs : c.ks)[to + (lane >> 2)] = (uint16_t)(__float_as_uint(s) >> 16);
}

int check_rows(const Kv4& c, const void* k, const void* v, int dtype, int64_t rows, int64_t k_row, int64_t k_head,
               int64_t v_row, int64_t v_head, const void* where, const int32_t* starts, const int32_t* err) {
  FBFP_CHECK_ARG(k && v && where && err, "null pointer");
  FBFP_CHECK_ARG(dtype_ok(dtype), "bad dtype %d", dtype);
  FBFP_CHECK_ARG(rows >= 1 && rows < (1 << 30), "bad row count %lld", (long long)rows);
  FBFP_CHECK_ARG(starts || rows <= c.seqs, "%lld rows without starts for %d sequences", (long long)rows, c.seqs);
  FBFP_CHECK_ARG(k_row >= 0 && k_head >= 0 && v_row >= 0 && v_head >= 0, "negative stride");
  FBFP_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & (dtype_size(dtype) - 1)) == 0, "rows must be aligned to their type");
  return FBFP_OK;
}

bool rows_vec(const void* k, const void* v, int dtype, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head) {
  const int64_t per = 16 / dtype_size(dtype);
  return (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((k_row | k_head | v_row | v_head) & (per - 1)) == 0;
}

// Rows of a thread: eight (four of fp32) where that still gives each SM eight CTAs, four where it gives it three,
// else one. Measured, write and read together, with 1 / 2 / 4 / 8 rows: 2048 rows x 8 heads x 256 of bf16 19.7 /
// 17.3 / 16.5 / 19.5 us; 131016 rows x 8 heads x 128 of fp16 read 285 / 173 / 131 / 116 us (5.95 TB/s).
template <typename T, bool VEC, int NG>
int launch_rows(bool write, void* stream, const Kv4& c, const RowsArg& r, const int32_t* at, const int32_t* starts,
                int32_t* err) {
  const Shape sh = shape_of(2 * c.nkv * 4 * NG);
  constexpr int kMost = sizeof(T) == 4 ? 4 : 8;
  const int64_t work = r.rows * sh.parts;
  const int rows = work >= (int64_t)148 * 8 * kMost * sh.rows ? kMost : work >= (int64_t)148 * 3 * 4 * sh.rows ? 4 : 1;
  auto kernel = write ? (rows == kMost ? kv4_write_kernel<T, VEC, NG, kMost>
                         : rows == 4   ? kv4_write_kernel<T, VEC, NG, 4> : kv4_write_kernel<T, VEC, NG, 1>)
                      : (rows == kMost ? kv4_read_kernel<T, VEC, NG, kMost>
                         : rows == 4   ? kv4_read_kernel<T, VEC, NG, 4> : kv4_read_kernel<T, VEC, NG, 1>);
  const int64_t per = (int64_t)sh.rows * rows;
  FBFP_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)((r.rows + per - 1) / per), sh.parts), dim3(kThreads), 0,
                           as_stream(stream), c, r, sh, at, starts, err));
  FBFP_LAUNCH_CHECK(write ? "kv4_write_kernel" : "kv4_read_kernel");
  return FBFP_OK;
}
template <typename T, bool VEC>
int launch_groups(bool write, void* stream, const Kv4& c, const RowsArg& r, const int32_t* at, const int32_t* starts,
                  int32_t* err) {
  switch (c.groups) {
    case 1: return launch_rows<T, VEC, 1>(write, stream, c, r, at, starts, err);
    case 2: return launch_rows<T, VEC, 2>(write, stream, c, r, at, starts, err);
    case 3: return launch_rows<T, VEC, 3>(write, stream, c, r, at, starts, err);
    case 4: return launch_rows<T, VEC, 4>(write, stream, c, r, at, starts, err);
    case 5: return launch_rows<T, VEC, 5>(write, stream, c, r, at, starts, err);
    case 6: return launch_rows<T, VEC, 6>(write, stream, c, r, at, starts, err);
    case 7: return launch_rows<T, VEC, 7>(write, stream, c, r, at, starts, err);
    default: return launch_rows<T, VEC, 8>(write, stream, c, r, at, starts, err);
  }
}
int launch_any(bool write, int dtype, bool vec, void* stream, const Kv4& c, const RowsArg& r, const int32_t* at,
               const int32_t* starts, int32_t* err) {
  if (dtype == FBFP_BF16)
    return vec ? launch_groups<__nv_bfloat16, true>(write, stream, c, r, at, starts, err)
               : launch_groups<__nv_bfloat16, false>(write, stream, c, r, at, starts, err);
  if (dtype == FBFP_F16)
    return vec ? launch_groups<__half, true>(write, stream, c, r, at, starts, err)
               : launch_groups<__half, false>(write, stream, c, r, at, starts, err);
  return vec ? launch_groups<float, true>(write, stream, c, r, at, starts, err)
             : launch_groups<float, false>(write, stream, c, r, at, starts, err);
}

}  // namespace
}  // namespace fbfp

using namespace fbfp;

extern "C" int fbfp_kv4_write(const fbfp_kv4_cache* cache, const void* k, const void* v, int dtype, int64_t rows,
                              int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head, const int32_t* pos,
                              const int32_t* starts, int32_t* err, void* stream) {
  Kv4 c;
  int st = kv4_check(cache, c);
  if (!st) st = check_rows(c, k, v, dtype, rows, k_row, k_head, v_row, v_head, pos, starts, err);
  if (st) return st;
  const bool vec = rows_vec(k, v, dtype, k_row, k_head, v_row, v_head);
  const RowsArg r{k, v, k_row, k_head, v_row, v_head, rows};
  return launch_any(true, dtype, vec, stream, c, r, pos, starts, err);
}

extern "C" int fbfp_kv4_read(const fbfp_kv4_cache* cache, void* k, void* v, int dtype, int64_t rows, int64_t k_row,
                             int64_t k_head, int64_t v_row, int64_t v_head, const int32_t* first,
                             const int32_t* starts, int32_t* err, void* stream) {
  Kv4 c;
  int st = kv4_check(cache, c);
  if (!st) st = check_rows(c, k, v, dtype, rows, k_row, k_head, v_row, v_head, first, starts, err);
  if (st) return st;
  const bool vec = rows_vec(k, v, dtype, k_row, k_head, v_row, v_head);
  const RowsArg r{k, v, k_row, k_head, v_row, v_head, rows};
  return launch_any(false, dtype, vec, stream, c, r, first, starts, err);
}

extern "C" int fbfp_kv4_append(const fbfp_kv4_cache* cache, const void* qkv, int64_t rows, int64_t heads,
                               const void* q_norm_w, const void* k_norm_w, float eps, const void* cos_table,
                               const void* sin_table, const int32_t* pos, const int32_t* starts, void* q_out,
                               int32_t* err, void* stream) {
  Kv4 c;
  int st = kv4_check(cache, c);
  if (st) return st;
  FBFP_CHECK_ARG(qkv && q_norm_w && k_norm_w && cos_table && sin_table && pos && q_out && err, "null pointer");
  FBFP_CHECK_ARG(c.hd % 16 == 0, "head_dim %d is not a multiple of 16", c.hd);
  FBFP_CHECK_ARG(heads >= 1 && heads <= 65535 && heads % c.nkv == 0, "%lld heads over %d", (long long)heads, c.nkv);
  FBFP_CHECK_ARG(rows >= 1 && rows < (1 << 30), "bad row count %lld", (long long)rows);
  FBFP_CHECK_ARG(starts || rows <= c.seqs, "%lld rows without starts for %d sequences", (long long)rows, c.seqs);
  if (((uintptr_t)qkv | (uintptr_t)q_norm_w | (uintptr_t)k_norm_w | (uintptr_t)cos_table | (uintptr_t)sin_table |
       (uintptr_t)q_out) & 15)
    return set_error(FBFP_ERR_ALIGN, "rows, weights and tables must be 16-byte aligned");
  const int64_t warps = rows * (heads + 2 * c.nkv), blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
  FBFP_CHECK_ARG(blocks <= 0x7FFFFFFF, "too many rows");
  typedef const __nv_bfloat16* P;
  FBFP_CUDA_TRY(launch_pdl(kv4_append_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, as_stream(stream), c, (P)qkv,
                           rows, (int)heads, (P)q_norm_w, (P)k_norm_w, eps, (P)cos_table, (P)sin_table, pos, starts,
                           (__nv_bfloat16*)q_out, err));
  FBFP_LAUNCH_CHECK("kv4_append_kernel");
  return FBFP_OK;
}
