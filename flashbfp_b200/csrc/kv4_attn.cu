// kv4_attn.cu — attention of the newest tokens over the 4-bit cache: one CTA per (row, query head), a
// warp per key in turn, an online softmax per warp, merged at the end.
#include "kv4.cuh"
#include "pdl.cuh"

namespace fbfp {
namespace {

constexpr int kWarps = 8;

struct CachedKeys {
  Kv4 c;
  int b, h;
  __device__ __forceinline__ void load(const uint8_t* v, const uint16_t* s, int64_t j, int lane, float (&x)[8]) const {
    const int64_t at = c.at(b, h, j) * c.groups;
    if (lane * 8 < c.hd) {
      kv4_values(reinterpret_cast<const uint32_t*>(v + at * 16)[lane], bf16_bits_to_float(s[at + (lane >> 2)]), x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
  }
  __device__ __forceinline__ void key(int64_t j, int lane, float (&x)[8]) const { load(c.kv, c.ks, j, lane, x); }
  __device__ __forceinline__ void value(int64_t j, int lane, float (&x)[8]) const { load(c.vv, c.vs, j, lane, x); }
};

template <typename T, typename Keys>
__device__ void attend_row(const T* q, T* out, int hd, const Keys& keys, int64_t lo, int64_t hi, float scaling) {
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int code = std::is_same<T, __half>::value ? FBFP_F16 : FBFP_BF16;
  float qv[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    qv[i] = lane * 8 < hd ? load_as_float(q + lane * 8, code, i) : 0.f;
    o[i] = 0.f;
  }
  for (int64_t j = lo + warp; j < hi; j += kWarps) {
    float x[8], s = 0.f;
    keys.key(j, lane, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += qv[i] * x[i];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= scaling;
    const float mn = fmaxf(m, s);
    const float f = __expf(m - mn), p = __expf(s - mn);
    m = mn;
    l = l * f + p;
    keys.value(j, lane, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * f + p * x[i];
  }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][lane * 8 + i] = o[i];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < kWarps; ++w) L += sm[w] == -INFINITY ? 0.f : sl[w] * __expf(sm[w] - M);
  for (int d = threadIdx.x; d < hd; d += blockDim.x) {
    float a = 0.f;
    for (int w = 0; w < kWarps; ++w) a += sm[w] == -INFINITY ? 0.f : so[w][d] * __expf(sm[w] - M);
    store_from_float(out, code, d, L > 0.f ? a / L : 0.f);
  }
}

struct Kv4Args {
  const void* q;
  void* out;
  int64_t q_seq, q_row, q_head, o_seq, o_row, o_head, window;
  int rows, heads;
  const int32_t* pos;
  int32_t* err;
  float scaling;
};

template <typename T>
__global__ void kv4_rows_kernel(Kv4 c, Kv4Args a) {
  pdl_prologue();
  const int h = (int)(blockIdx.x % a.heads), kvh = h / (a.heads / c.nkv);
  const int r = (int)(blockIdx.x / a.heads), b = r / a.rows, i = r % a.rows;
  int64_t at = (int64_t)a.pos[b] + i;
  if (at < 0 || at >= c.positions) {
    if (threadIdx.x == 0) atomicExch(a.err, 2);
    at = -1;
  }
  const int64_t lo = a.window > 0 ? max(at - a.window + 1, (int64_t)0) : 0;
  CachedKeys keys{c, b, kvh};
  attend_row((const T*)a.q + b * a.q_seq + i * a.q_row + h * a.q_head,
             (T*)a.out + b * a.o_seq + i * a.o_row + h * a.o_head, c.hd, keys, lo, at + 1, a.scaling);
}

}  // namespace
}  // namespace fbfp

using namespace fbfp;

extern "C" int64_t fbfp_kv4_attention_workspace_bytes(const fbfp_kv4_cache* cache, int64_t rows, int64_t heads) {
  return 0;
}

extern "C" int fbfp_kv4_attention(const fbfp_kv4_cache* cache, const void* q, int dtype, int64_t rows, int64_t heads,
                                  int64_t q_seq, int64_t q_row, int64_t q_head, const int32_t* pos, int64_t window,
                                  float scaling, void* out, int64_t o_seq, int64_t o_row, int64_t o_head,
                                  void* workspace, int64_t workspace_bytes, int32_t* err, void* stream) {
  Kv4 c;
  const int st = kv4_check(cache, c);
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
  Kv4Args a{q, out, q_seq, q_row, q_head, o_seq, o_row, o_head, window, (int)rows, (int)heads, pos, err, scaling};
  FBFP_CHECK_ARG(c.seqs * rows * heads <= 0x7FFFFFFF, "too many rows");
  auto kernel = dtype == FBFP_BF16 ? kv4_rows_kernel<__nv_bfloat16> : kv4_rows_kernel<__half>;
  FBFP_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)(c.seqs * rows * heads)), dim3(kWarps * 32), 0, as_stream(stream), c, a));
  FBFP_LAUNCH_CHECK("kv4_rows_kernel");
  return FBFP_OK;
}
