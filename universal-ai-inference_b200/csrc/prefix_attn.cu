// prefix_attn.cu -- attention of new tokens over a prefix that the whole batch shares and each sequence's own
// cached positions, straight from an f16 or 8-bit cache (formats: kv_cache.cu).
//
//   s_j = scale * ks_j * (q . c_j),   out = sum_j e^(s_j - m) vs_j c'_j / sum_j e^(s_j - m)
//
// with c_j, c'_j the stored K and V values of position j and ks_j, vs_j their row scales (1 for f16).
// Token t of sequence b sees prefix positions [0, P) and own positions [0, own_len[b] - T + t]; a row that sees
// none is zero.  Running maximum, sums and outputs are f32.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cfloat>

#include "serve_kernels.hpp"

namespace uaii_b200 {
namespace {

template <int F, int N>
__device__ __forceinline__ void load_values(const void* row, int lane, float (&x)[N]) {
  if constexpr (F == kKvF16) {
    const __half* p = static_cast<const __half*>(row) + N * lane;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __half2float(p[i]);
  } else {
    const uint8_t* p = static_cast<const uint8_t*>(row) + N * lane;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (F == kKvI8) x[i] = (float)((int)p[i] - 128);
      else x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)p[i], __NV_E4M3)));
    }
  }
}

// One warp per query row, one cached position at a time.
template <int F, int HD, typename Q>
__global__ void __launch_bounds__(128) prefix_attn_row_kernel(PrefixAttnArgs a) {
  constexpr int N = HD / 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= a.B * a.T * a.H) return;
  const int64_t h = row % a.H, t = (row / a.H) % a.T, b = row / (a.H * a.T);
  const int64_t kvh = h / (a.H / a.own.heads);
  const Q* qp = static_cast<const Q*>(a.q) + b * a.qs.batch + t * a.qs.token + h * a.qs.head + N * lane;
  float q[N], o[N] = {}, m = -FLT_MAX, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = (float)qp[i] * a.scale;
  int64_t len = a.own_len[b];
  if (len < 0 || len > a.own.max_seq) {
    if (lane == 0) atomicExch(a.err, kErrKvLength);
    len = len < 0 ? 0 : a.own.max_seq;
  }
  for (int part = a.prefix.k ? 0 : 1; part < 2; ++part) {
    const KvCache& c = part ? a.own : a.prefix;
    const int64_t base = (part ? b * c.heads + kvh : kvh) * c.max_seq;
    const int64_t n = part ? len - a.T + t + 1 : a.prefix_len;
    constexpr int kBytes = F == kKvF16 ? 2 * HD : HD;
    for (int64_t j = 0; j < n; ++j) {
      float x[N], s = 0.f;
      load_values<F>(static_cast<const char*>(c.k) + (base + j) * kBytes, lane, x);
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(q[i], x[i], s);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (F != kKvF16) s *= c.k_scale[base + j];
      const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
      m = mn;
      l = fmaf(l, f, p);
      load_values<F>(static_cast<const char*>(c.v) + (base + j) * kBytes, lane, x);
      const float pv = F == kKvF16 ? p : p * c.v_scale[base + j];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(o[i], f, pv * x[i]);
    }
  }
  Q* out = static_cast<Q*>(a.out) + row * HD + N * lane;
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (Q)(l > 0.f ? o[i] / l : 0.f);
}

template <int F, typename Q>
void run_rows(const PrefixAttnArgs& a, cudaStream_t st) {
  const unsigned g = (unsigned)((a.B * a.T * a.H + 3) / 4);
  if (a.own.hd == 128) prefix_attn_row_kernel<F, 128, Q><<<g, 128, 0, st>>>(a);
  else prefix_attn_row_kernel<F, 64, Q><<<g, 128, 0, st>>>(a);
}

template <typename Q>
void run_fmt(const PrefixAttnArgs& a, cudaStream_t st) {
  if (a.own.fmt == kKvI8) run_rows<kKvI8, Q>(a, st);
  else if (a.own.fmt == kKvE4M3) run_rows<kKvE4M3, Q>(a, st);
  else run_rows<kKvF16, Q>(a, st);
}

}  // namespace

size_t prefix_attn_ws(const PrefixAttnArgs&) { return 0; }

cudaError_t launch_prefix_attn(const PrefixAttnArgs& a, void*, int* launches, cudaStream_t st) {
  if (a.half) run_fmt<__half>(a, st);
  else run_fmt<float>(a, st);
  *launches = 1;
  return cudaGetLastError();
}

}  // namespace uaii_b200
