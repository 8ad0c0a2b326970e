// kv_cache.cu -- the KV cache written (quantised as it is written) and read back.
//
// A row is the head_dim values x of one (sequence, kv head, position) of K or of V.  With a = max|x|:
//   i8    scale = a / 127, byte = 128 + rint(x * (127 / a)), value = (byte - 128) * scale
//   e4m3  scale = a / 448, byte = e4m3(x * (448 / a)),       value = e4m3^-1(byte) * scale
// One scale for a whole row keeps the bytes exact operands of f16 tensor-core products: the scale of a
// position leaves the sum over head_dim in q.k and joins the probability in p.v.  Rows with a < 2^-100
// (whose reciprocal would overflow) become zeros; a row with an infinity or a NaN gets a NaN scale, so the
// fault shows wherever the row is used instead of turning into finite values.  Every step is one IEEE
// operation, so the bytes are the same on every run and equal the formula's.
//
// Both kernels are bound by the bytes they move: one pass, 16-byte accesses, nothing kept between rows.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "serve_kernels.hpp"

namespace uaii_b200 {
namespace {

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr int kRows = 2;  // rows of a thread, loaded together

__device__ __forceinline__ void load8(const float* p, bool vec, float (&x)[8]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ void load8(const __half* p, bool vec, float (&x)[8]) {
  __half h[8];
  if (vec) {
    *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __half2float(h[i]);
}

// HD / 8 lanes hold a row, 8 consecutive values each, and store it at `row` unless that is null (every lane of the
// warp takes part in the maxima); returns the row's scale (0 for f16, which has none).
template <int F, int HD>
__device__ __forceinline__ float store_row8(const float (&x)[8], void* row, int lane8) {
  if constexpr (F == kKvF16) {
    __half h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = __float2half_rn(x[i]);
    if (row) reinterpret_cast<uint4*>(row)[lane8] = *reinterpret_cast<const uint4*>(h);
    return 0.f;
  } else {
    // |x| as bits: an infinity or a NaN compares above every finite value
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float top = F == kKvI8 ? 127.f : 448.f, amax = __uint_as_float(a);
    const bool fine = a < 0x7f800000u && amax >= kTiny;
    const float inv = fine ? __fdiv_rn(top, amax) : 0.f;
    uint32_t w[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = fine ? __fmul_rn(x[4 * p + i], inv) : 0.f;
        if constexpr (F == kKvI8) b[i] = (uint32_t)(__float2int_rn(y) + 128);
        else b[i] = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
      }
      w[p] = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
    }
    if (row) reinterpret_cast<uint2*>(row)[lane8] = make_uint2(w[0], w[1]);
    return a >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fine ? __fdiv_rn(amax, top) : 0.f;
  }
}

// One group of HD / 8 lanes per row: grid (tokens x heads of a sequence, heads fastest; sequence; K or V), kRows groups
// of heads x tokens a block apart for each thread, their loads under way together.
template <int F, int HD, typename X>
__global__ void __launch_bounds__(256) kv_append_kernel(KvCache c, const X* __restrict__ k, const X* __restrict__ v,
                                                        int T, RowView s, const int32_t* __restrict__ pos,
                                                        const int32_t* __restrict__ n_new, bool vec, int* err) {
  constexpr int kLanes = HD / 8, kGroups = 256 / kLanes;
  const int lane8 = threadIdx.x % kLanes, heads = (int)c.heads, b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const X* from = (is_v ? v : k) + b * s.batch + 8 * lane8;
  const int count = n_new ? min(n_new[b], T) : T, start = pos[b], rows = count * heads;
  char* out = static_cast<char*>(is_v ? c.v : c.k);
  float* scales = is_v ? c.v_scale : c.k_scale;
  constexpr int kBytes = F == kKvF16 ? 2 * HD : HD;
  float x[kRows][8] = {};
  int64_t row[kRows];  // of the cache; -1: none
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = (blockIdx.x * kRows + i) * kGroups + threadIdx.x / kLanes, t = r / heads, h = r - t * heads;
    const int64_t at = (int64_t)start + t;
    row[i] = -1;
    if (r >= rows) continue;
    if (at < 0 || at >= c.max_seq) {
      if (lane8 == 0) atomicExch(err, kErrKvPosition);
      continue;
    }
    row[i] = ((int64_t)b * heads + h) * c.max_seq + at;
    load8(from + t * s.token + h * s.head, vec, x[i]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float sc = store_row8<F, HD>(x[i], row[i] >= 0 ? out + row[i] * kBytes : nullptr, lane8);
    if (F != kKvF16 && row[i] >= 0 && lane8 == 0) scales[row[i]] = sc;
  }
}

template <int F>
__device__ __forceinline__ float value_of(uint32_t byte, float scale) {
  if constexpr (F == kKvI8) return __fmul_rn((float)((int)byte - 128), scale);
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
  return __fmul_rn(__half2float(__half(h)), scale);
}

__device__ __forceinline__ void put8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void put8(__half* p, const float (&x)[8]) {
  __half h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = __float2half_rn(x[i]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// Positions of one (sequence, head) plane, K or V: grid (positions; plane; K or V).  A thread takes 16 values of a row,
// kRows rows a block apart.
template <int F, int HD, typename Y>
__global__ void __launch_bounds__(256) kv_read_kernel(KvCache c, int64_t pos0, int n, Y* __restrict__ k_out, Y* __restrict__ v_out) {
  constexpr int kLanes = HD / 16, kGroups = 256 / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool is_v = blockIdx.z != 0;
  const int64_t plane = (int64_t)blockIdx.y * c.max_seq + pos0;
  const char* from = static_cast<const char*>(is_v ? c.v : c.k);
  const float* scales = is_v ? c.v_scale : c.k_scale;
  Y* to = (is_v ? v_out : k_out) + (int64_t)blockIdx.y * n * HD + 16 * lane;
  constexpr int kLoads = F == kKvF16 ? 2 : 1;  // of 16 bytes
  uint4 w[kRows][kLoads];
  float sc[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int j = (blockIdx.x * kRows + i) * kGroups + threadIdx.x / kLanes;
    sc[i] = 0.f;
    if (j >= n) continue;
    const uint4* src = reinterpret_cast<const uint4*>(from + (plane + j) * (HD * kLoads)) + lane * kLoads;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) w[i][l] = __ldcs(src + l);
    if (F != kKvF16) sc[i] = __ldcs(scales + plane + j);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int j = (blockIdx.x * kRows + i) * kGroups + threadIdx.x / kLanes;
    if (j >= n) continue;
    float x[2][8];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const uint4 q = w[i][F == kKvF16 ? k / 8 : 0];
      if constexpr (F == kKvF16) {
        const int e = k & 7;
        const uint32_t u = e < 2 ? q.x : e < 4 ? q.y : e < 6 ? q.z : q.w;
        x[k / 8][e] = __half2float(__ushort_as_half((unsigned short)(e & 1 ? u >> 16 : u & 0xffffu)));
      } else {
        const uint32_t u = k < 4 ? q.x : k < 8 ? q.y : k < 12 ? q.z : q.w;
        x[k / 8][k & 7] = value_of<F>((u >> (8 * (k & 3))) & 255u, sc[i]);
      }
    }
    put8(to + (int64_t)j * HD, x[0]);
    put8(to + (int64_t)j * HD + 8, x[1]);
  }
}

template <int F, typename X>
cudaError_t append_fmt(const KvCache& c, const X* k, const X* v, int64_t T, const RowView& s, const int32_t* pos,
                       const int32_t* n_new, int* err, cudaStream_t st) {
  const int64_t per = kRows * (256 / (c.hd / 8)), blocks = (T * c.heads + per - 1) / per;
  if (blocks > 0x7fffffff || c.batch > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)c.batch, 2);
  const size_t m = 16 / sizeof(X);  // 16-byte loads where every row starts on such a boundary
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 && s.batch % m == 0 &&
                   s.token % m == 0 && s.head % m == 0;
  if (c.hd == 128) kv_append_kernel<F, 128, X><<<grid, 256, 0, st>>>(c, k, v, (int)T, s, pos, n_new, vec, err);
  else kv_append_kernel<F, 64, X><<<grid, 256, 0, st>>>(c, k, v, (int)T, s, pos, n_new, vec, err);
  return cudaGetLastError();
}

template <typename X>
cudaError_t append_any(const KvCache& c, const void* k, const void* v, int64_t T, const RowView& s, const int32_t* pos,
                       const int32_t* n_new, int* err, cudaStream_t st) {
  const X *a = static_cast<const X*>(k), *b = static_cast<const X*>(v);
  if (c.fmt == kKvI8) return append_fmt<kKvI8>(c, a, b, T, s, pos, n_new, err, st);
  if (c.fmt == kKvE4M3) return append_fmt<kKvE4M3>(c, a, b, T, s, pos, n_new, err, st);
  return append_fmt<kKvF16>(c, a, b, T, s, pos, n_new, err, st);
}

template <int F, typename Y>
cudaError_t read_fmt(const KvCache& c, int64_t pos0, int64_t n, Y* k, Y* v, cudaStream_t st) {
  const int64_t per = kRows * (256 / (c.hd / 16)), blocks = (n + per - 1) / per;
  if (c.batch * c.heads > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)(c.batch * c.heads), 2);
  if (c.hd == 128) kv_read_kernel<F, 128, Y><<<grid, 256, 0, st>>>(c, pos0, (int)n, k, v);
  else kv_read_kernel<F, 64, Y><<<grid, 256, 0, st>>>(c, pos0, (int)n, k, v);
  return cudaGetLastError();
}

template <typename Y>
cudaError_t read_any(const KvCache& c, int64_t pos0, int64_t n, void* k, void* v, cudaStream_t st) {
  Y *a = static_cast<Y*>(k), *b = static_cast<Y*>(v);
  if (c.fmt == kKvI8) return read_fmt<kKvI8>(c, pos0, n, a, b, st);
  if (c.fmt == kKvE4M3) return read_fmt<kKvE4M3>(c, pos0, n, a, b, st);
  return read_fmt<kKvF16>(c, pos0, n, a, b, st);
}

}  // namespace

cudaError_t launch_kv_append(const KvCache& c, const void* k, const void* v, bool half, int64_t T, const RowView& s,
                             const int32_t* pos, const int32_t* n_new, int* err, cudaStream_t st) {
  return half ? append_any<__half>(c, k, v, T, s, pos, n_new, err, st)
              : append_any<float>(c, k, v, T, s, pos, n_new, err, st);
}

cudaError_t launch_kv_read(const KvCache& c, int64_t pos0, int64_t n, void* k_out, void* v_out, bool half,
                           cudaStream_t st) {
  return half ? read_any<__half>(c, pos0, n, k_out, v_out, st) : read_any<float>(c, pos0, n, k_out, v_out, st);
}

}  // namespace uaii_b200
