// sample.cu -- one token per row of logits from a given uniform number, with temperature, top-k, top-p and min-p.
//
// With m = max l and e_i = exp((l_i - m) / temperature), tokens are ranked by logit, the lower index first among
// equals.  Kept are the first top_k of the ranking, of those the shortest leading part whose mass reaches top_p of
// theirs, and of those the tokens with e_i >= min_p (the first in the ranking always).  The token is the first kept
// index whose running mass over the kept indices, in index order, exceeds floor(u * mass(kept)).
//
// Masses are whole numbers, w_i = rint(e_i * 2^31), summed in 64 bits: every order of summation gives the same sums,
// so neither the split over threads nor the order of shared-memory atomics can change the token.  Sampling in index
// order (not in rank order) draws from the same distribution and needs no sort: the kept set is all logits above a
// threshold and the first few that equal it, and a radix descent over the logits' ordered bits finds the threshold.
#include <cuda_fp16.h>

#include "serve_kernels.hpp"

namespace uaii_b200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 256;

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const __half* p) { return __half2float(*p); }

// Ordered bits of a logit: larger keys for larger logits, one key for both zeros; a NaN counts as -inf.
__device__ __forceinline__ uint32_t key_of_logit(float x) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float weight_exp(float x, float m, float heat) {
  return x == m ? 1.0f : expf(__fdiv_rn(__fsub_rn(x, m), heat));
}
__device__ __forceinline__ uint64_t weight(float e) { return (uint64_t)__float2ull_rn(__fmul_rn(e, 2147483648.0f)); }

struct Cut {
  uint32_t key;   // kept: keys above it, and the first `ties` indices whose key equals it
  uint64_t ties;
};

struct Shared {
  uint64_t hist[kBins];
  uint64_t scan[32];
  uint32_t digit;
  uint64_t above;
};

__device__ uint64_t block_sum64(uint64_t v, Shared& s) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
  for (int i = 0; i < kThreads / 32; ++i) t += s.scan[i];
  return t;
}

__device__ uint64_t block_exclusive64(uint64_t v, Shared& s) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint64_t inc = v;
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();
  if (lane == 31) s.scan[w] = inc;
  __syncthreads();
  uint64_t before = 0;
  for (int i = 0; i < w; ++i) before += s.scan[i];
  return before + inc - v;
}

// The smallest leading part of the ranking whose size (a count of tokens, or their mass) reaches `goal` > 0: four
// passes of eight bits, each adding the tokens that share the digits found so far into 256 bins.
template <bool MASS, typename X>
__device__ Cut find_cut(const X* row, int64_t V, float m, float heat, uint64_t goal, Shared& s) {
  uint32_t prefix = 0;
  uint64_t above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.hist[i] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < V; i += kThreads) {
      const float x = logit(row + i);
      const uint32_t k = key_of_logit(x);
      if (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
      const uint64_t add = MASS ? weight(weight_exp(logit_of_key(k), m, heat)) : 1;
      if (add) atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[(k >> shift) & 255]), (unsigned long long)add);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t sum = above;
      int d = kBins - 1;
      for (; d > 0 && sum + s.hist[d] < goal; --d) sum += s.hist[d];
      s.digit = (uint32_t)d;
      s.above = sum;
    }
    __syncthreads();
    prefix |= s.digit << shift;
    above = s.above;
  }
  const uint64_t each = MASS ? weight(weight_exp(logit_of_key(prefix), m, heat)) : 1;
  return Cut{prefix, each ? (goal - above + each - 1) / each : 1};
}

template <typename X>
__global__ void __launch_bounds__(kThreads) sample_kernel(const X* __restrict__ logits, int64_t V, int64_t ld,
                                                          const float* __restrict__ temperature,
                                                          const int32_t* __restrict__ top_k,
                                                          const float* __restrict__ top_p,
                                                          const float* __restrict__ min_p, const float* __restrict__ u,
                                                          int32_t* __restrict__ tokens, float* __restrict__ probs,
                                                          int32_t* __restrict__ kept) {
  __shared__ Shared s;
  const int64_t b = blockIdx.x;
  const X* row = logits + b * ld;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x; i < V; i += kThreads) top = max(top, key_of_logit(logit(row + i)));
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; ++i) top = max(top, (uint32_t)s.scan[i]);
  __syncthreads();
  const float m = logit_of_key(top);
  if (m == -INFINITY) {  // no token has any mass
    if (threadIdx.x == 0) {
      tokens[b] = -1;
      if (probs) probs[b] = 0.f;
      if (kept) kept[b] = 0;
    }
    return;
  }
  const float heat_in = temperature[b];
  const bool greedy = !(heat_in > 0.f);
  const float heat = greedy ? 1.0f : heat_in;
  const int64_t k = greedy ? 1 : top_k[b];
  const float p = top_p[b], least = min_p[b];
  Cut cut{0, 0};
  bool cut_set = false;
  if (k > 0 && k < V) {
    cut = k == 1 ? Cut{top, 1} : find_cut<false>(row, V, m, heat, (uint64_t)k, s);
    cut_set = true;
  }
  if (!(p >= 1.0f) && k != 1) {
    uint64_t mass = 0;
    for (int64_t i = threadIdx.x; i < V; i += kThreads) {
      const uint32_t key = key_of_logit(logit(row + i));
      if (key > cut.key || !cut_set) mass += weight(weight_exp(logit_of_key(key), m, heat));
    }
    mass = block_sum64(mass, s);
    if (cut_set) mass += cut.ties * weight(weight_exp(logit_of_key(cut.key), m, heat));
    const double want = ceil((double)p * (double)mass);
    const uint64_t reach = want > 0.0 ? (uint64_t)want : 0;  // p <= 0 or NaN: the first token alone
    cut = reach ? find_cut<true>(row, V, m, heat, reach, s) : Cut{top, 1};
    cut_set = true;
  }
  if (!(least <= 1.0f)) {  // min_p above 1 or NaN: the first token alone
    cut = Cut{top, 1};
    cut_set = true;
  }
  const float e_tie = cut_set ? weight_exp(logit_of_key(cut.key), m, heat) : 0.f;
  const uint64_t w_tie = weight(e_tie), tie_max = cut.key == top || e_tie >= least ? cut.ties : 0;
  // 1 and e: kept above the cut; 2: equals it
  auto side = [&](uint32_t key, float& e) {
    if (cut_set && key <= cut.key) return key == cut.key ? 2 : 0;
    e = weight_exp(logit_of_key(key), m, heat);
    return e >= least ? 1 : 0;
  };
  // kept mass and ties of each thread's run of indices
  const int64_t run = (V + kThreads - 1) / kThreads, i0 = min(V, run * threadIdx.x), i1 = min(V, i0 + run);
  uint64_t mass = 0, ties = 0, count = 0;
  for (int64_t i = i0; i < i1; ++i) {
    float e = 0.f;
    const int f = side(key_of_logit(logit(row + i)), e);
    if (f == 1) {
      mass += weight(e);
      ++count;
    }
    ties += f == 2;
  }
  const uint64_t ties_before = block_exclusive64(ties, s);
  const uint64_t my_ties = min(ties_before + ties, tie_max) - min(ties_before, tie_max);
  mass += my_ties * w_tie;
  count += my_ties;
  const uint64_t before = block_exclusive64(mass, s);
  const uint64_t total = block_sum64(mass, s);
  const uint64_t n_kept = block_sum64(count, s);
  const double w = floor((double)u[b] * (double)total);
  uint64_t goal = w > 0.0 ? (uint64_t)w : 0;
  if (goal >= total) goal = total - 1;
  if (before <= goal && goal < before + mass) {  // this thread's run holds the token
    uint64_t sum = before, t = ties_before;
    for (int64_t i = i0; i < i1; ++i) {
      float e = 0.f;
      const int f = side(key_of_logit(logit(row + i)), e);
      uint64_t add = f == 1 ? weight(e) : 0;
      if (f == 2) add = t++ < tie_max ? w_tie : 0;
      sum += add;
      if (sum > goal) {
        tokens[b] = (int32_t)i;
        if (probs) probs[b] = (float)((double)add / (double)total);
        if (kept) kept[b] = (int32_t)n_kept;
        break;
      }
    }
  }
}

}  // namespace

cudaError_t launch_sample(const void* logits, bool half, int64_t B, int64_t V, int64_t ld, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tokens,
                          float* probs, int32_t* kept, cudaStream_t st) {
  if (half)
    sample_kernel<<<(unsigned)B, kThreads, 0, st>>>(static_cast<const __half*>(logits), V, ld, temperature, top_k,
                                                    top_p, min_p, u, tokens, probs, kept);
  else
    sample_kernel<<<(unsigned)B, kThreads, 0, st>>>(static_cast<const float*>(logits), V, ld, temperature, top_k,
                                                    top_p, min_p, u, tokens, probs, kept);
  return cudaGetLastError();
}

}  // namespace uaii_b200
