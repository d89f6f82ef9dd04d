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

// One thread per 8 values of a row: (row, keys or values, head, piece), pieces innermost.
struct Piece {
  int64_t row;
  int which, head, piece;
};
__device__ __forceinline__ Piece piece_of(int64_t i, int nkv, int per_head) {
  const uint32_t per_row = 2u * nkv * per_head;
  Piece q;
  q.row = i / per_row;
  uint32_t rest = (uint32_t)(i - q.row * per_row);
  q.piece = rest % per_head;
  rest /= per_head;
  q.which = rest >= (uint32_t)nkv;
  q.head = rest - (q.which ? nkv : 0);
  return q;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(Kv4 c, RowsArg r, const int32_t* pos,
                                                             const int32_t* starts, int32_t* err) {
  pdl_prologue();
  const int per_head = 4 * c.groups;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const Piece q = piece_of(i, c.nkv, per_head);
  int b = -1;
  int64_t at = 0;
  if (q.row < r.rows) {
    b = packed_seq(q.row, starts, c.seqs, at);
    if (b >= 0) at += pos[b];
    if (b >= 0 && (at < 0 || at >= c.positions)) {
      if (q.piece == 0) atomicExch(err, 2);
      b = -1;
    }
  }
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (b >= 0 && q.piece * 8 < c.hd) {
    const T* p = q.which ? (const T*)r.v + q.row * r.v_row + q.head * r.v_head
                         : (const T*)r.k + q.row * r.k_row + q.head * r.k_head;
    load8<T, VEC>(p + q.piece * 8, x);
  }
  uint32_t word;
  float s;
  kv4_quantise(x, word, s);
  if (b < 0) return;
  const int64_t to = c.at(b, q.head, at) * c.groups;
  reinterpret_cast<uint32_t*>((q.which ? c.vv : c.kv) + to * 16)[q.piece] = word;
  if ((q.piece & 3) == 0) (q.which ? c.vs : c.ks)[to + (q.piece >> 2)] = (uint16_t)(__float_as_uint(s) >> 16);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4 c, RowsArg r, const int32_t* first,
                                                            const int32_t* starts, int32_t* err) {
  pdl_prologue();
  const int per_head = c.hd / 8;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const Piece q = piece_of(i, c.nkv, per_head);
  if (q.row >= r.rows) return;
  int64_t at;
  const int b = packed_seq(q.row, starts, c.seqs, at);
  if (b < 0) return;
  at += first[b];
  if (at < 0 || at >= c.positions) {
    if (q.piece == 0) atomicExch(err, 2);
    return;
  }
  const int64_t from = c.at(b, q.head, at) * c.groups;
  const uint32_t word = reinterpret_cast<const uint32_t*>((q.which ? c.vv : c.kv) + from * 16)[q.piece];
  const float s = bf16_bits_to_float((q.which ? c.vs : c.ks)[from + (q.piece >> 2)]);
  float x[8];
  kv4_values(word, s, x);
  T* p = q.which ? (T*)r.v + q.row * r.v_row + q.head * r.v_head : (T*)r.k + q.row * r.k_row + q.head * r.k_head;
  store8<T, VEC>(p + q.piece * 8, x);
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
    if (lane == 0) atomicExch(err, 2);
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
  kv4_quantise(x, word, s);
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

template <typename K>
int launch_rows(K kernel, int64_t threads, void* stream, const Kv4& c, const RowsArg& r, const int32_t* at,
                const int32_t* starts, int32_t* err) {
  const int64_t blocks = (threads + kThreads - 1) / kThreads;
  FBFP_CHECK_ARG(blocks <= 0x7FFFFFFF, "too many rows");
  FBFP_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, as_stream(stream), c, r, at, starts, err));
  return FBFP_OK;
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
  auto kernel = dtype == FBFP_BF16 ? (vec ? kv4_write_kernel<__nv_bfloat16, true> : kv4_write_kernel<__nv_bfloat16, false>)
                : dtype == FBFP_F16 ? (vec ? kv4_write_kernel<__half, true> : kv4_write_kernel<__half, false>)
                                    : (vec ? kv4_write_kernel<float, true> : kv4_write_kernel<float, false>);
  st = launch_rows(kernel, rows * 2 * c.nkv * 4 * c.groups, stream, c, r, pos, starts, err);
  if (st) return st;
  FBFP_LAUNCH_CHECK("kv4_write_kernel");
  return FBFP_OK;
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
  auto kernel = dtype == FBFP_BF16 ? (vec ? kv4_read_kernel<__nv_bfloat16, true> : kv4_read_kernel<__nv_bfloat16, false>)
                : dtype == FBFP_F16 ? (vec ? kv4_read_kernel<__half, true> : kv4_read_kernel<__half, false>)
                                    : (vec ? kv4_read_kernel<float, true> : kv4_read_kernel<float, false>);
  st = launch_rows(kernel, rows * 2 * c.nkv * (c.hd / 8), stream, c, r, first, starts, err);
  if (st) return st;
  FBFP_LAUNCH_CHECK("kv4_read_kernel");
  return FBFP_OK;
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
