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
// Both kernels make one pass and keep nothing between rows.  Prompts of 4096 tokens and fewer, 8 heads of 128, f16 to e4m3
// and back to f16: the append of 12450 tokens (77 MB) 22.8 us, 3.4 TB/s, 0.52 of a copy's rate (16 values a thread, since
// index, maximum and two divisions cost a thread as much as the conversions; with 8 values 29.5 us), the read of 4 x 4096
// (102 MB) 13.5 us, the bytes partly still in L2.  16 values
// a thread made the read slower (20 against 13.5 us): its stores then lie 32 bytes apart.  A token or two is bound by
// the launch.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <type_traits>

#include "serve_kernels.hpp"

namespace uaii_b200 {
namespace {

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr int kRows = 2, kReadRows = 4;  // rows of a thread, loaded together

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

__device__ __forceinline__ float larger(float a, float b) {  // a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// HD / 16 lanes hold a row, of each half 8 values in a row, and store it at `row` unless that is null (every lane of the
// warp takes part in the maxima); returns the row's scale (0 for f16, which has none).
template <int F, int HD>
__device__ __forceinline__ float store_row(const float (&x)[2][8], char* row, int lane) {
  if constexpr (F == kKvF16) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      __half h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = __float2half_rn(x[d][i]);
      if (row) reinterpret_cast<uint4*>(row + d * HD)[lane] = *reinterpret_cast<const uint4*>(h);
    }
    return 0.f;
  } else {
    float amax = 0.f;
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = larger(amax, fabsf(x[d][i]));
#pragma unroll
    for (int o = HD / 32; o > 0; o >>= 1) amax = larger(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float top = F == kKvI8 ? 127.f : 448.f;
    const bool fine = amax >= kTiny && amax < INFINITY;
    const float inv = __fdiv_rn(top, amax);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      uint32_t w[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __fmul_rn(x[d][4 * p + i], inv);
        if constexpr (F == kKvI8) {  // added to 3 * 2^22 + 128, a number rounds to a whole one whose low byte is the code
          uint32_t u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(__fadd_rn(y[i], 12583040.0f));
          w[p] = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
        } else {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
          w[p] = lo | (hi << 16);
        }
        if (!fine) w[p] = F == kKvI8 ? 0x80808080u : 0u;
      }
      if (row) reinterpret_cast<uint2*>(row + d * (HD / 2))[lane] = make_uint2(w[0], w[1]);
    }
    if (lane != 0) return 0.f;
    return fine ? __fdiv_rn(amax, top) : amax < INFINITY ? 0.f : __uint_as_float(0x7fffffffu);
  }
}

// One group of HD / 16 lanes per row: grid (tokens x heads of a sequence, heads fastest; sequence; K or V), kRows groups
// of heads x tokens a block apart for each thread, their loads under way together.
template <int F, int HD, typename X>
__global__ void __launch_bounds__(256) kv_append_kernel(KvCache c, const X* __restrict__ k, const X* __restrict__ v,
                                                        int T, RowView s, const int32_t* __restrict__ pos,
                                                        const int32_t* __restrict__ n_new, bool vec, int s_t, int s_h,
                                                        int* err) {
  constexpr int kLanes = HD / 16, kGroups = 256 / kLanes;  // (kGroups = s_t * heads + s_h)
  const int lane = threadIdx.x % kLanes, heads = (int)c.heads, b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const X* from = (is_v ? v : k) + b * s.batch + 8 * lane;
  const int count = n_new ? min(n_new[b], T) : T, start = pos[b], rows = count * heads;
  char* out = static_cast<char*>(is_v ? c.v : c.k);
  float* scales = is_v ? c.v_scale : c.k_scale;
  constexpr int kBytes = F == kKvF16 ? 2 * HD : HD;
  float x[kRows][2][8] = {};
  int64_t row[kRows];  // of the cache; -1: none
  int r = blockIdx.x * kRows * kGroups + threadIdx.x / kLanes, t = r / heads, h = r - t * heads;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (i) {
      r += kGroups;
      h += s_h;
      t += s_t;
      if (h >= heads) {
        h -= heads;
        ++t;
      }
    }
    const int64_t at = (int64_t)start + t;
    row[i] = -1;
    if (r >= rows) continue;
    if (at < 0 || at >= c.max_seq) {
      if (lane == 0) atomicExch(err, kErrKvPosition);
      continue;
    }
    row[i] = ((int64_t)b * heads + h) * c.max_seq + at;
    const X* src = from + t * s.token + h * s.head;
    load8(src, vec, x[i][0]);
    load8(src + HD / 2, vec, x[i][1]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float sc = store_row<F, HD>(x[i], row[i] >= 0 ? out + row[i] * kBytes : nullptr, lane);
    if (F != kKvF16 && row[i] >= 0 && lane == 0) scales[row[i]] = sc;
  }
}

// Bytes 2 p and 2 p + 1 of w as values.
template <int F>
__device__ __forceinline__ float2 values_of(uint32_t w, int p, float scale) {
  float2 y;
  if constexpr (F == kKvI8) {  // a byte behind 0x4b0000 is the float 2^23 + byte
    y.x = __uint_as_float(__byte_perm(w, 0x4b000000u, p ? 0x7442 : 0x7440)) - 8388736.0f;
    y.y = __uint_as_float(__byte_perm(w, 0x4b000000u, p ? 0x7443 : 0x7441)) - 8388736.0f;
  } else {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * p) & 0xffffu), __NV_E4M3);
    y = __half22float2(__half2(h));
  }
  return make_float2(__fmul_rn(y.x, scale), __fmul_rn(y.y, scale));
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

// Positions of one (sequence, head) plane, K or V: grid (positions; plane; K or V).  A thread takes 8 values of a row (so
// that a warp's 16-byte stores of f16 lie side by side), kReadRows rows a block apart, their loads under way together.
template <int F, int HD, typename Y>
__global__ void __launch_bounds__(256) kv_read_kernel(KvCache c, int64_t pos0, int n, Y* __restrict__ k_out, Y* __restrict__ v_out) {
  constexpr int kLanes = HD / 8, kGroups = 256 / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool is_v = blockIdx.z != 0;
  const int64_t plane = (int64_t)blockIdx.y * c.max_seq + pos0;
  const char* from = static_cast<const char*>(is_v ? c.v : c.k);
  const float* scales = is_v ? c.v_scale : c.k_scale;
  Y* to = (is_v ? v_out : k_out) + (int64_t)blockIdx.y * n * HD + 8 * lane;
  using Word = std::conditional_t<F == kKvF16, uint4, uint2>;
  Word w[kReadRows];
  float sc[kReadRows];
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const int j = (blockIdx.x * kReadRows + i) * kGroups + threadIdx.x / kLanes;
    sc[i] = 0.f;
    if (j >= n) continue;
    w[i] = __ldcs(reinterpret_cast<const Word*>(from + (plane + j) * (HD / 8 * (int)sizeof(Word))) + lane);
    if (F != kKvF16) sc[i] = __ldcs(scales + plane + j);
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const int j = (blockIdx.x * kReadRows + i) * kGroups + threadIdx.x / kLanes;
    if (j >= n) continue;
    float x[8];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      float2 y;
      if constexpr (F == kKvF16) {
        const uint32_t u = p == 0 ? w[i].x : p == 1 ? w[i].y : p == 2 ? w[i].z : w[i].w;
        y = __half22float2(__halves2half2(__ushort_as_half((unsigned short)(u & 0xffffu)), __ushort_as_half((unsigned short)(u >> 16))));
      } else {
        y = values_of<F>(p < 2 ? w[i].x : w[i].y, p & 1, sc[i]);
      }
      x[2 * p] = y.x;
      x[2 * p + 1] = y.y;
    }
    put8(to + (int64_t)j * HD, x);
  }
}

template <int F, typename X>
cudaError_t append_fmt(const KvCache& c, const X* k, const X* v, int64_t T, const RowView& s, const int32_t* pos,
                       const int32_t* n_new, int* err, cudaStream_t st) {
  const int64_t per = kRows * (256 / (c.hd / 16)), blocks = (T * c.heads + per - 1) / per;
  if (blocks > 0x7fffffff || c.batch > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)c.batch, 2);
  const size_t m = 16 / sizeof(X);  // 16-byte loads where every row starts on such a boundary
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 && s.batch % m == 0 &&
                   s.token % m == 0 && s.head % m == 0;
  const int groups = 256 / (c.hd / 16), s_t = groups / (int)c.heads, s_h = groups % (int)c.heads;
  if (c.hd == 128) kv_append_kernel<F, 128, X><<<grid, 256, 0, st>>>(c, k, v, (int)T, s, pos, n_new, vec, s_t, s_h, err);
  else kv_append_kernel<F, 64, X><<<grid, 256, 0, st>>>(c, k, v, (int)T, s, pos, n_new, vec, s_t, s_h, err);
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
  const int64_t per = kReadRows * (256 / (c.hd / 8)), blocks = (n + per - 1) / per;
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
