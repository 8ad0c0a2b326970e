// sample.cu -- one token per row of logits from a given uniform number, with temperature, top-k, top-p and min-p.
//
// With m = max l and e_i = exp((l_i - m) / temperature), tokens are ranked by logit, the lower index first among
// equals.  Kept are the first top_k of the ranking, of those the shortest leading part whose mass reaches top_p of
// theirs, and of those the tokens with e_i >= min_p (the first in the ranking always).  The token is the first kept
// index whose running mass over the kept indices, in index order, exceeds floor(u * mass(kept)).
//
// Masses are whole numbers, w_i = rint(e_i * 2^31), summed in 64 bits: every order of summation gives the same sums,
// so neither the split over threads nor the order of shared-memory atomics can change the token.  Sampling in index
// order (not in rank order) draws from the same distribution and needs no sort: a weight never falls as its logit
// rises, so the kept set is all weights above a cut, and of the weights that equal it the first few by logit and index.
//
// A cluster of up to eight CTAs holds a row: every logit is read once and its weight kept in shared memory.  The cut is
// found with one histogram over the weights' leading bits and a ranking, by logit, of the few tokens of one bin; counts,
// sums and bins of the CTAs meet through distributed shared memory.
// 256 rows of 151936 f16 logits take 273 us (77 MB read once, which alone would be 12 us): 127 instructions a logit at
// 0.55 of the issue rate, with two CTAs an SM; of a CTA's 60000 cycles 10000 go to reading, 7000 to weights, 8000 to the
// histogram's atomics, 7000 to ranking, 6000 to the kept mass and 15000 to cluster barriers.  A single row takes
// 20 us on the device: passes over a few logits a thread and cluster barriers, one after the other.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "serve_kernels.hpp"

namespace cg = cooperative_groups;

namespace uaii_b200 {
namespace {

constexpr uint32_t kOne = 1u << 31;  // the weight of the largest logit

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const __half* p) { return __half2float(*p); }

// A NaN counts as -inf (the maximum of a NaN and a number is the number), and both zeros are one.
__device__ __forceinline__ float canonical(float x) { return fmaxf(x, -INFINITY) + 0.0f; }
// Ordered bits of a canonical logit: larger keys for larger logits.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint32_t key_of_logit(float x) { return key_of(canonical(x)); }
__device__ __forceinline__ float logit_of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint32_t weight(float e) { return __float2uint_rn(__fmul_rn(e, 2147483648.0f)); }

// exp((x - m) / heat), each step rounded once, for x <= m.
struct Heat {
  float m, h, r;
  bool plain;  // h far from the ends of the range
  // Correctly rounded quotient by a divisor used often, from its correctly rounded reciprocal and fused residuals
  // (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  Quotients so
  // small that a residual would round are below the last place of the exponential's argument 0 anyway.
  __device__ __forceinline__ float quotient(float a, float q) const {
    q = fmaf(fmaf(-q, h, a), r, q);
    return fmaf(fmaf(-q, h, a), r, q);
  }
  __device__ __forceinline__ float exp_of(float x) const {
    if (x == m) return 1.0f;
    const float a = __fsub_rn(x, m);
    return expf(plain ? quotient(a, __fmul_rn(a, r)) : __fdiv_rn(a, h));
  }
  // The weight.  In the plain range without a branch; below e^-24 it is 0, whatever the exponential of the product.
  template <bool PLAIN>
  __device__ __forceinline__ uint32_t weight_in(float x) const {
    if constexpr (PLAIN) {
      const float a = __fsub_rn(x, m), q = __fmul_rn(a, r);
      const uint32_t y = weight(expf(quotient(a, q)));
      return x == m ? kOne : q < -24.0f ? 0 : y;
    }
    return weight(exp_of(x));
  }
  __device__ __forceinline__ uint32_t weight_of(float x) const { return plain ? weight_in<true>(x) : weight_in<false>(x); }
};

// One row's settings.
struct Setting {
  bool greedy;
  float heat, p, least, u;
  int64_t k;
};
__device__ __forceinline__ Setting setting_of(int64_t b, const float* temperature, const int32_t* top_k, const float* top_p,
                                              const float* min_p, const float* u) {
  Setting s;
  const float t = temperature[b];
  s.greedy = !(t > 0.f);
  s.heat = s.greedy ? 1.0f : t;
  s.k = top_k[b];
  s.p = top_p[b];
  s.least = min_p[b];
  s.u = u[b];
  if (s.greedy || !(s.least <= 1.0f)) s.k = 1;  // the first token alone
  return s;
}

__device__ __forceinline__ uint64_t target_of(float u, uint64_t total) {
  const double w = floor((double)u * (double)total);
  const uint64_t goal = w > 0.0 ? (uint64_t)w : 0;
  return goal < total ? goal : total - 1;
}
__device__ __forceinline__ uint64_t reach_of(float p, uint64_t mass) {  // at least 1: the first token is always kept
  const double want = ceil((double)p * (double)mass);
  return want > 1.0 ? (uint64_t)want : 1;
}

// ---------------------------------------------------------------- a row in a cluster's shared memory

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 512, kList = 1024, kMaxCluster = 8;
constexpr int kGroups = kThreads / (kBins / 2);         // threads that read the same bins, of different CTAs
constexpr int kFixed = (2 + kGroups) * kBins * 8 + 2 * kList * 4;  // dynamic shared memory besides the weights
constexpr int kMaxSlice = (int)(kSampleMaxVocab / kMaxCluster);  // weights of a CTA
static_assert(kList <= kGroups * kBins, "the lists of all CTAs take the place of the sums");
static_assert(kFixed + 4 * kMaxSlice <= 225 * 1024, "a CTA's shared memory");

// Leading bits of a weight above 0: its exponent and four bits more, as f32 has them.
__device__ __forceinline__ int bin_of(uint32_t w) { return (int)(__float_as_uint(__uint2float_rz(w)) >> 19) - 127 * 16; }

struct Found {        // a cut: weights above `w` are kept, and `need` of the `equal` ones at it
  uint32_t w;
  uint64_t need, equal;
  bool ranked;        // those whose logit is above `edge`, and the first `ties` with that logit; else it is to be found
  uint32_t edge;
  uint64_t ties;
};

struct RowShared {
  uint64_t warp[kWarps];
  uint64_t part[5][kMaxCluster];  // numbers of each CTA, a row for each purpose
  int bin;                        // where the goal falls: the bin, and what lies above it
  uint64_t above;
  uint32_t listed[2];             // weights of that bin
  Found found;
  uint64_t segment[kWarps], ties[kWarps];
};
enum Purpose { kTop, kMass, kSome, kHead, kTail };

// What the CTAs of a cluster add up is read by each of them for itself, so that one cluster barrier is enough: bins and
// lists come in two sets, used in turn, and a set is written again only after the barrier of the other's use.
template <typename X>
struct Row {
  cg::cluster_group cluster;
  RowShared& sh;
  uint32_t* w;          // this CTA's weights, in index order; zeros up to a multiple of four
  uint32_t* bins;       // [2][2 kBins]: a bin's sums of low and of high halves (32-bit atomics are native)
  uint64_t* sums;       // [kGroups][kBins]
  uint32_t* list;       // [2][kList] indices of this CTA's tokens
  uint2* all;           // [kList] weights and keys of the tokens that all CTAs listed
  const X* x;           // the row's logits
  int slice;            // of which a CTA has so many
  int quads;            // fours of weights of this CTA
  int rank, ctas;
  int set;
  Heat heat;

  template <typename F>
  __device__ __forceinline__ void each4(F&& f) const {  // f(index, weight) in fours, whole CTA
    for (int q = threadIdx.x; q < quads; q += kThreads) f(4 * q, reinterpret_cast<const uint4*>(w)[q]);
  }
  __device__ __forceinline__ uint64_t block_sum(uint64_t v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < kWarps; ++i) t += sh.warp[i];
    return t;
  }
  // Publish this CTA's number to every CTA's array (a cluster barrier has to follow).
  __device__ __forceinline__ void tell(Purpose p, uint64_t v) {
    if ((int)threadIdx.x < ctas) cluster.map_shared_rank(sh.part[p], threadIdx.x)[rank] = v;
  }
  __device__ __forceinline__ uint64_t sum_of(Purpose p) const {
    uint64_t t = 0;
    for (int i = 0; i < ctas; ++i) t += sh.part[p][i];
    return t;
  }
  __device__ __forceinline__ uint32_t* next_bins() {
    set ^= 1;
    for (int i = threadIdx.x; i < kBins; i += kThreads) reinterpret_cast<uint2*>(bins + 2 * set * kBins)[i] = make_uint2(0, 0);
    if (threadIdx.x == 0) sh.listed[set] = 0;
    __syncthreads();
    return bins + 2 * set * kBins;
  }
  // Where a bin's low sum lies (the high one beside it, at ^ 1): every other sixteen bins the other way round, so that
  // low sums fall into all banks.
  static __device__ __forceinline__ int low_at(int bin) { return 2 * bin + (bin >> 4 & 1); }
  // The bin, from the highest down, at which the cluster's bins reach `goal`: sh.bin and sh.above (plus `above`).  Remote
  // shared memory gave 4 to 5 bytes a cycle to an SM, so bins are read in 512-byte pieces and are no more than
  // 512: 1024 took 4 us more, 256 left longer lists to rank (a tenth more at 256 rows of 151936).
  __device__ __forceinline__ void reach(uint64_t goal, uint64_t above) {
    constexpr int kEach = kMaxCluster / kGroups;
    const int t = threadIdx.x, at = t % (kBins / 2), group = t / (kBins / 2);
    uint4 y[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      y[k] = make_uint4(0, 0, 0, 0);
      const int c = k * kGroups + group;
      if (c < ctas) y[k] = reinterpret_cast<const uint4*>(cluster.map_shared_rank(bins + 2 * set * kBins, c))[at];
    }
    uint64_t two[2] = {};
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const bool turned = at & 8;
      two[0] += (turned ? y[k].y : y[k].x) + ((uint64_t)(turned ? y[k].x : y[k].y) << 16);
      two[1] += (turned ? y[k].w : y[k].z) + ((uint64_t)(turned ? y[k].z : y[k].w) << 16);
    }
    sums[group * kBins + 2 * at] = two[0];
    sums[group * kBins + 2 * at + 1] = two[1];
    __syncthreads();
    uint64_t mine = 0;
    if (t < kBins)
#pragma unroll
      for (int k = 0; k < kGroups; ++k) mine += sums[k * kBins + kBins - 1 - t];
    uint64_t inc = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if ((t & 31) >= o) inc += v;
    }
    if ((t & 31) == 31) sh.warp[t >> 5] = inc;
    __syncthreads();
    uint64_t before = above + inc - mine;
    for (int i = 0; i < (t >> 5); ++i) before += sh.warp[i];
    if (before < goal && goal <= before + mine) {
      sh.bin = kBins - 1 - t;
      sh.above = before;
    }
    __syncthreads();
  }

  __device__ __forceinline__ void put(uint32_t i) {  // token i of this CTA into its list
    const uint32_t k = atomicAdd(&sh.listed[set], 1u);
    if (k < kList) list[set * kList + k] = i;
  }
  // Of the tokens that the CTAs have listed, ranked by weight and then by logit (read again: should the exponential not
  // rise with its argument to the last bit, the ranking is still the one that the cut is applied by), the cut at which
  // the leading ones reach `goal`, `above` lying above them all.  False, with their count in f->equal, if they are more
  // than a list holds.
  template <bool MASS>
  __device__ bool rank_listed(uint64_t goal, uint64_t above, Found* f) {
    const int t = threadIdx.x;
    cluster.sync();
    uint32_t count[kMaxCluster], listed = 0;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) count[c] = c < ctas ? cluster.map_shared_rank(&sh, c)->listed[set] : 0;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) listed += count[c];
    f->equal = listed;
    if (listed > kList) return false;
    for (uint32_t i = t; i < listed; i += kThreads) {
      uint32_t j = i;
      int c = 0;
#pragma unroll
      for (int k = 0; k + 1 < kMaxCluster; ++k)
        if (c == k && j >= count[k]) {
          j -= count[k];
          c = k + 1;
        }
      const float y = canonical(logit(x + (int64_t)c * slice + cluster.map_shared_rank(list + set * kList, c)[j]));
      all[i] = make_uint2(heat.weight_of(y), key_of_logit(y));
    }
    __syncthreads();
    for (uint32_t i = t; i < listed; i += kThreads) {
      const uint2 me = all[i];
      uint64_t over = above;
      uint32_t same = 0, equal = 0, before = 0;  // of the same logit; of the same weight, and those with a larger logit
      for (uint32_t j = 0; j < listed; ++j) {
        const uint2 y = all[j];
        const bool level = y.x == me.x, higher = level && y.y > me.y;
        over += y.x > me.x || higher ? (MASS ? y.x : 1u) : 0u;
        same += y.y == me.y;
        equal += level;
        before += higher;
      }
      const uint64_t each = MASS ? me.x : 1;
      if (over < goal && goal <= over + same * each) {  // (equal tokens write the same)
        const uint64_t ties = (goal - over + each - 1) / each;
        sh.found = Found{me.x, before + ties, equal, true, me.y, ties};
      }
    }
    __syncthreads();
    *f = sh.found;
    __syncthreads();
    return true;
  }

  // The cut at which the leading weights reach `goal` (in tokens, or in mass).  `least`: weights below it cannot matter.
  template <bool MASS>
  __device__ Found find(uint64_t goal, uint32_t least) {
    // weights in [lo, hi] are binned: by leading bits at first, then, should a bin hold more than the list does, by
    // equal parts of its range
    uint32_t lo = least ? least : 1, hi = kOne;
    int shift = -1;
    uint64_t above = 0;
    for (;;) {
      uint32_t* mine = next_bins();
      auto bin = [&](auto&& of) {
        each4([&](int, uint4 v) {
          if (max(max(v.x, v.y), max(v.z, v.w)) < lo) return;
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int to = low_at(of(x[j]));
            if (x[j] >= lo && x[j] <= hi) {  // (50000 halves of 16 bits add up to less than 2^32)
              atomicAdd(mine + to, MASS ? x[j] & 0xffffu : 1u);
              if (MASS) atomicAdd(mine + (to ^ 1), x[j] >> 16);
            }
          }
        });
      };
      if (shift < 0) bin([](uint32_t y) { return bin_of(y); });
      else bin([&](uint32_t y) { return (int)((y - lo) >> shift); });
      cluster.sync();
      reach(goal, above);
      const int at = sh.bin;
      above = sh.above;
      uint32_t from, to;  // the bin's weights
      if (shift < 0) {
        const int e = at >> 4;
        from = e >= 4 ? (uint32_t)(16 + (at & 15)) << (e - 4) : (uint32_t)(16 + (at & 15)) >> (4 - e);
        to = e >= 4 ? from + ((1u << (e - 4)) - 1) : from;
      } else {
        from = lo + ((uint32_t)at << shift);
        to = from + ((1u << shift) - 1);
      }
      from = max(from, lo);
      to = min(to, hi);
      // the bin's weights
      each4([&](int i, uint4 v) {
        if (max(max(v.x, v.y), max(v.z, v.w)) < from) return;
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (x[j] >= from && x[j] <= to) put(i + j);
      });
      Found f;
      if (rank_listed<MASS>(goal, above, &f)) return f;
      if (from == to) return Found{from, MASS ? (goal - above + from - 1) / from : goal - above, f.equal, false, 0, 0};
      lo = from;
      hi = to;
      const int bits = 32 - __clz(to - from);
      shift = bits > 9 ? bits - 9 : 0;
    }
  }
};

template <typename X>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const X* __restrict__ logits, int64_t V, int64_t ld, int slice, bool vec,
                                                          const float* __restrict__ temperature,
                                                          const int32_t* __restrict__ top_k,
                                                          const float* __restrict__ top_p,
                                                          const float* __restrict__ min_p, const float* __restrict__ u,
                                                          int32_t* __restrict__ tokens, float* __restrict__ probs,
                                                          int32_t* __restrict__ kept) {
  extern __shared__ uint4 dynamic[];
  __shared__ RowShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // this CTA has started: the others may write to its shared memory once all have
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int64_t b = blockIdx.x / ctas, begin = (int64_t)rank * slice;
  const int n = (int)max(int64_t(0), min((int64_t)slice, V - begin));
  uint32_t* bins = reinterpret_cast<uint32_t*>(dynamic);
  uint64_t* sums = reinterpret_cast<uint64_t*>(bins + 4 * kBins);
  uint2* all = reinterpret_cast<uint2*>(sums);  // the one in use while the other is not
  uint32_t* list = reinterpret_cast<uint32_t*>(sums + kGroups * kBins);
  uint32_t* w = list + 2 * kList;
  const X* x = logits + b * ld + begin;
  Row<X> row{cluster, sh, w, bins, sums, list, all, logits + b * ld, slice, (n + 3) / 4, rank, ctas, 0, {}};
  const Setting s = setting_of(b, temperature, top_k, top_p, min_p, u);

  // the logits, read once, and their largest
  float most = -INFINITY;
  constexpr int kVec = 16 / sizeof(X);
  const int whole = vec ? n / kVec * kVec : 0;
#pragma unroll 4
  for (int i = t * kVec; i < whole; i += kThreads * kVec) {
    X v[kVec];
    *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(x + i));
    float f[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      f[j] = canonical((float)v[j]);
      most = fmaxf(most, f[j]);
    }
#pragma unroll
    for (int j = 0; j < kVec; j += 4) *reinterpret_cast<float4*>(w + i + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
  }
  for (int i = whole + t; i < n; i += kThreads) {
    const float f = canonical(logit(x + i));
    most = fmaxf(most, f);
    w[i] = __float_as_uint(f);
  }
  if (n + t < 4 * row.quads) w[n + t] = 0xff800000u;  // -inf
  uint32_t top = key_of(most);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) sh.warp[warp] = top;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) top = max(top, (uint32_t)sh.warp[i]);
  cluster.barrier_wait();  // (the reading hid it)
  row.tell(kTop, top);
  cluster.sync();
  for (int i = 0; i < ctas; ++i) top = max(top, (uint32_t)sh.part[kTop][i]);
  const float m = logit_of_key(top);
  if (m == -INFINITY) {  // no token has any mass (the same in every CTA)
    if (rank == 0 && t == 0) {
      tokens[b] = -1;
      if (probs) probs[b] = 0.f;
      if (kept) kept[b] = 0;
    }
    return;
  }

  // weights in place of the logits
  const Heat heat = row.heat = {m, s.heat, __fdiv_rn(1.0f, s.heat), s.heat >= 0x1p-30f && s.heat <= 0x1p30f};
  uint64_t mass = 0;
  uint32_t some = 0;
  auto weigh = [&](auto plain) {
    row.each4([&](int i, uint4 v) {
      const uint4 y = {heat.template weight_in<plain.value>(__uint_as_float(v.x)), heat.template weight_in<plain.value>(__uint_as_float(v.y)),
                       heat.template weight_in<plain.value>(__uint_as_float(v.z)), heat.template weight_in<plain.value>(__uint_as_float(v.w))};
      *reinterpret_cast<uint4*>(w + i) = y;
      mass += ((uint64_t)y.x + y.y) + ((uint64_t)y.z + y.w);
      some += (y.x != 0) + (y.y != 0) + (y.z != 0) + (y.w != 0);
    });
  };
  if (heat.plain) weigh(std::true_type{});
  else weigh(std::false_type{});
  mass = row.block_sum(mass);
  some = (uint32_t)row.block_sum(some);
  row.tell(kMass, mass);
  row.tell(kSome, some);
  cluster.sync();
  mass = row.sum_of(kMass);
  const uint64_t positive = row.sum_of(kSome);

  // the cut: none (w 0), or weights above cut.w and `need` of the `equal` ones at it
  Found cut{};
  const bool by_count = s.k > 0 && s.k < V;
  if (s.k == 1) {
    cut = Found{kOne, 1, 2, true, top, 1};  // the first of the largest
  } else if (by_count && (uint64_t)s.k < positive) {
    cut = row.template find<false>((uint64_t)s.k, 0);
  }
  if (!(s.p >= 1.0f) && s.k != 1) {
    uint64_t z = mass;
    if (cut.w) {  // the mass of the first k
      uint64_t v = 0;
      row.each4([&](int, uint4 y) {
        v += ((uint64_t)(y.x > cut.w ? y.x : 0) + (y.y > cut.w ? y.y : 0)) + ((uint64_t)(y.z > cut.w ? y.z : 0) + (y.w > cut.w ? y.w : 0));
      });
      row.tell(kHead, row.block_sum(v));
      cluster.sync();
      z = row.sum_of(kHead) + cut.need * cut.w;
    }
    const uint64_t goal = reach_of(s.p, z);
    // Weights below (z - goal) / V add up to less than z - goal: the goal is reached above them.
    cut = row.template find<true>(goal, (uint32_t)max((z - goal) / (uint64_t)V, (uint64_t)cut.w));
  }
  const bool partial = cut.w != 0 && cut.need < cut.equal;
  uint32_t edge = cut.edge;
  uint64_t ties = cut.ties;
  if (partial && !cut.ranked) {  // more equal weights than a list holds: eight bits of their keys at a time
    uint64_t need = cut.need;
    for (int shift = 24; shift >= 0; shift -= 8) {
      uint32_t* mine = row.next_bins();
      row.each4([&](int i, uint4 v) {
        const uint32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (y[j] != cut.w) continue;
          const uint32_t k = key_of_logit(logit(x + i + j));
          if (shift == 24 || (k >> (shift + 8)) == (edge >> (shift + 8))) atomicAdd(mine + row.low_at((k >> shift) & 255), 1u);
        }
      });
      cluster.sync();
      row.reach(need, 0);
      edge |= (uint32_t)sh.bin << shift;
      need -= sh.above;
      __syncthreads();
    }
    ties = need;
  }

  // Kept or not: 1 kept, 2 at the edge (kept if among the first `ties` there), 0 not.  A weight equal to min_p's, which
  // rounding may have brought there from below, is told by its exponential.
  const float least = s.k == 1 ? 0.f : s.least;
  const uint32_t w_least = least > 0.f ? weight(least) : 0;
  auto side = [&](int i, uint32_t y) {
    if (i >= n) return 0;
    if (y < cut.w || y < w_least) return 0;
    if (least > 0.f && y == w_least && !(heat.exp_of(canonical(logit(x + i))) >= least)) return 0;
    if (y > cut.w || !partial) return 1;
    const uint32_t k = key_of_logit(logit(x + i));
    return k > edge ? 1 : k == edge ? 2 : 0;
  };
  // masses and ties of each warp's run of indices, four of them a lane
  const uint32_t low = max(cut.w, w_least);
  const int run = (row.quads + kWarps - 1) / kWarps, q0 = min(row.quads, run * warp), q1 = min(row.quads, q0 + run);
  const bool cuts = cut.w != 0 || least > 0.f;
  uint64_t seg_mass = 0;
  uint32_t seg_ties = 0, seg_count = 0;
  for (int q = q0 + lane; q < q1; q += 32) {
    const uint4 v = reinterpret_cast<const uint4*>(w)[q];
    // above both cuts a token is kept, at one of them it takes a look (without a cut none does: zeros have no mass)
    bool look = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t y = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
      seg_mass += y > low ? y : 0;
      seg_count += y > low;
      look |= y == low;
    }
    if (look && cuts) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t y = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
        if (y != low) continue;
        const int f = side(4 * q + j, y);
        seg_mass += f == 1 ? y : 0;
        seg_count += f == 1;
        seg_ties += f == 2;
      }
    }
  }
  for (int o = 16; o > 0; o >>= 1) seg_mass += __shfl_xor_sync(0xffffffffu, seg_mass, o);
  seg_ties = __reduce_add_sync(0xffffffffu, seg_ties);
  seg_count = __reduce_add_sync(0xffffffffu, seg_count);
  if (lane == 0) {
    sh.segment[warp] = seg_mass;
    sh.ties[warp] = seg_ties;
  }
  const uint64_t cta_count = row.block_sum(lane == 0 ? seg_count : 0);  // (its barriers also cover segment and ties)
  uint64_t cta_mass = 0, cta_ties = 0;
  for (int i = 0; i < kWarps; ++i) {
    cta_mass += sh.segment[i];
    cta_ties += sh.ties[i];
  }
  row.tell(kTail, cta_mass);
  row.tell(kTop, cta_ties | cta_count << 32);
  cluster.sync();
  uint64_t total = 0, all_count = 0, all_ties = 0, before = 0, ties_before = 0;
  for (int c = 0; c < ctas; ++c) {
    const uint64_t more = sh.part[kTop][c] & 0xffffffffu;
    if (c < rank) ties_before += more;
    const uint64_t in = min(all_ties + more, ties) - min(all_ties, ties), add = sh.part[kTail][c] + in * cut.w;
    if (c < rank) before += add;
    total += add;
    all_ties += more;
    all_count += (sh.part[kTop][c] >> 32) + in;
  }
  const uint64_t goal = target_of(s.u, total);
  if (rank == 0 && t == 0 && kept) {
    // tokens without mass count too, where nothing cuts them off
    uint64_t count = all_count;
    if (cut.w == 0 && !(least > 0.f)) count = by_count ? min((uint64_t)s.k, (uint64_t)V) : (uint64_t)V;
    else if (cut.w == 0 && by_count) count = min(count, (uint64_t)s.k);
    kept[b] = (int32_t)count;
  }
  for (int i = 0; i < warp; ++i) {
    const uint64_t more = sh.ties[i];
    before += sh.segment[i] + (min(ties_before + more, ties) - min(ties_before, ties)) * cut.w;
    ties_before += more;
  }
  const uint64_t mine = sh.segment[warp] + (min(ties_before + sh.ties[warp], ties) - min(ties_before, ties)) * cut.w;
  if (before <= goal && goal < before + mine) {  // this warp's run holds the token
    // a lane's part of it: a few fours in a row
    const int each = (q1 - q0 + 31) / 32, l0 = min(q1, q0 + each * lane), l1 = min(q1, l0 + each);
    uint64_t sum = 0;
    uint32_t edges = 0;
    for (int q = l0; q < l1; ++q) {
      const uint4 v = reinterpret_cast<const uint4*>(w)[q];
      if (max(max(v.x, v.y), max(v.z, v.w)) < low) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t y = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
        const int f = side(4 * q + j, y);
        sum += f == 1 ? y : 0;
        edges += f == 2;
      }
    }
    uint64_t inc = edges;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    ties_before += inc - edges;
    sum += (min(ties_before + edges, ties) - min(ties_before, ties)) * cut.w;
    inc = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    before += inc - sum;
    if (before <= goal && goal < before + sum) {
      for (int q = 4 * l0; before <= goal; ++q) {
        const int f = side(q, w[q]);
        const uint64_t add = f == 1 ? w[q] : f == 2 && ties_before++ < ties ? cut.w : 0;
        before += add;
        if (before > goal) {
          tokens[b] = (int32_t)(begin + q);
          if (probs) probs[b] = (float)((double)add / (double)total);
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_sample(const void* logits, bool half, int64_t B, int64_t V, int64_t ld, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tokens,
                          float* probs, int32_t* kept, cudaStream_t st) {
  const size_t esz = half ? 2 : 4;
  // CTAs of a row: 4096 logits each where that is enough, eight at most
  int ctas = 1;
  while (ctas < kMaxCluster && V > 4096 * (int64_t)ctas) ctas *= 2;
  const int64_t slice = ((V + ctas - 1) / ctas + 7) / 8 * 8;
  if (slice > kMaxSlice) return cudaErrorInvalidValue;
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && ld * (int64_t)esz % 16 == 0;
  const int smem = kFixed + (int)slice * 4;
  auto run = [&](auto kern, const auto* x) -> cudaError_t {
    // the limit of the kernel, not this call's: another backend's thread may be between its own two calls
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + 4 * kMaxSlice);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(B * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)ctas, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, x, V, ld, (int)slice, vec, temperature, top_k, top_p, min_p, u, tokens, probs, kept);
  };
  return half ? run(sample_kernel<__half>, static_cast<const __half*>(logits))
              : run(sample_kernel<float>, static_cast<const float*>(logits));
}

}  // namespace uaii_b200
