// attn_common.cuh -- what the attention kernels (attn_narrow.cuh, attn_wide.cuh) share: stored tiles and their bytes
// as f16 operands, items and pieces, and the CTAs' shares of the work.  The mathematics is in prefix_attn.cu.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "serve_kernels.hpp"
#include "umma.cuh"

namespace uaii_b200 {
namespace attn {

constexpr int kSms = 148;
constexpr int kTile = 64;        // wide: keys of a tile
constexpr int kWarps = 4;        // narrow: warps of a CTA
constexpr int kNarrowCtas = 3;   // narrow: CTAs per SM (wide: one)
constexpr int kMaxScan = 512;    // sequences whose unit counts a CTA sums itself
constexpr float kLog2e = 1.4426950408889634f;
// A position's weight is 2^(s - m + 9) in the denominator, and that times V's row scale (1 in an f16 cache) where it meets
// V's bytes.  Only the second becomes f16, so a row's reference m is a whole number at or above the largest product 2^s vs
// so far, not the largest score: a V row much larger than the others does not push them out of f16's range unless its
// product outweighs theirs.  (A reference made from the scales alone lost 2e-4 of a result beside a row 10^6 times
// larger whose own weight was 0, and all of it beside one 10^12 times larger.)  m moves only when a product has come to
// be near f16's end: the sums are then seldom rescaled, and the two f16 parts of a product (split_weights) are off by at most
// 2^-22 of it or 2^-32 of the largest, whichever is more.
// The denominator is f32 and may lie far from 1; V rows of scale 0, whose products ask for no reference, are held within
// it by kOver.
constexpr float kLift = 9.0f, kSlack = 6.0f, kOver = 96.0f;
constexpr float kMostProduct = 15.f, kMostWeight = 110.f;  // binary orders
constexpr float kLeastScale = 0x1p-96f;

// A stored row, and a copied tile of KEYS rows of K or V: boxes of at most 128 bytes a row (the swizzle span).
template <int F, int HD, int KEYS>
struct Tile {
  static constexpr int kEsz = F == kKvF16 ? 2 : 1;
  static constexpr int kRow = HD * kEsz;
  static constexpr int kPart = kRow < 128 ? kRow : 128;
  static constexpr int kBoxes = kRow / kPart;
  static constexpr int kBoxBytes = kPart * KEYS;
  static constexpr int kBytes = kBoxes * kBoxBytes;
  static constexpr int kScaleBytes = F == kKvF16 ? 0 : 2 * KEYS * 4;
};

struct Maps {
  CUtensorMap pk, pv, ok, ov;
};

// Division by a number that the host knows: n / d = floor(n m / 2^(31 + s)) for 0 <= n < 2^31, with 2^s >= d and
// m = ceil(2^(31 + s) / d) < 2^32 (m d exceeds 2^(31 + s) by less than d <= 2^s, n times that is below 2^(31 + s)).
// The plain operator took a worker's walk to its next piece 3500 cycles, most of it six divisions one after the other.
struct Div {
  uint32_t m = 0;
  int s = 0;  // 0: d = 1
  Div() = default;
  explicit Div(int d) {
    while ((int64_t(1) << s) < d) ++s;
    m = (uint32_t)(((uint64_t(1) << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d);
  }
};
__device__ __forceinline__ int operator/(int n, const Div& d) { return d.s ? (int)(__umulhi((uint32_t)n, d.m) >> (d.s - 1)) : n; }

// The items of one kernel: prefix items first, then own ones (either may be missing).
struct Plan {
  int G;                   // query heads per kv head
  int prefix_rows;         // B * T * G
  int own_rows;            // T * G
  int rt;                  // rows of an item
  int slot_rows, subs;     // rows of a slot; parts of an item's rows in it (2: each half of the keys has its own)
  bool split_keys;         // wide: the two row tiles hold the same rows
  int unit;                // keys of a unit
  int prefix_nrt, own_nrt; // items per kv head (0: none)
  int lead;                // units without keys at the start of every item, for what a piece costs beside its keys
  int prefix_units;        // units of a prefix item, the lead among them
  int prefix_items;
  int grid;                // CTAs (0: the kernel has no work)
  int workers;             // shares of the work: wide CTAs or narrow warps
  Div by_G, by_rt, by_own_rows, by_own_nrt, by_prefix_nrt, by_prefix_units, by_workers;
  float* part;             // partial sums [slot][slot_rows][hd]
  float* ml;               // (reference, denominator) of each partial row
};

__device__ __forceinline__ int own_length(const PrefixAttnArgs& a, int64_t b, bool report) {
  int64_t n = a.own_len[b];
  if (n < 0 || n > a.own.max_seq) {
    if (report) atomicExch(a.err, kErrKvLength);
    n = n < 0 ? 0 : a.own.max_seq;
  }
  return (int)n;
}

// ---------------------------------------------------------------- operands

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(  // not volatile: independent products may be interleaved
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2 of a V scale's size, to a tenth: an f32's bits as a number (straight lines between powers of two, never above it;
// 0 counts as 2^-127).
__device__ __forceinline__ float log2_scale(float vs) {
  return fmaf((float)(__float_as_int(vs) & 0x7fffffff), 0x1p-23f, -127.f);
}
// The reference after positions with this largest score and largest product: whole numbers, so that neither the factors nor
// the differences to them round.
__device__ __forceinline__ float next_reference(float m, float top, float product) {
  return fmaxf(fmaxf(m, ceilf(product)), ceilf(top) - kOver);
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// h, but the smallest half of s's sign rather than 0 unless s is 0.
__device__ __forceinline__ __half but_zero(__half h, float s) {
  return __hisnan(h) || (__half_as_ushort(h) & 0x7fff) || s == 0.f ? h : __ushort_as_half(s < 0.f ? 0x8001 : 1);
}

// Two weights as leading parts, cut off after f16's 11 bits, and what that left, rounded: off by at most 2^-22 of the weight
// or 2^-25, and below 2^-14, where the leading part is rounded again, by 2^-24.  (Rounding the leading part and taking the rest from its value makes a longer chain:
// 128 sequences behind 32801 positions took 130.8 us against 124.9.)  INFINITE: V may hold infinities and both parts meet
// it in one accumulator, so the rest is not 0 where there is a leading part (0 * inf is NaN).
template <bool INFINITE>
__device__ __forceinline__ void split_weights(float x, float y, uint32_t& lead, uint32_t& rest) {
  const float u = __uint_as_float(__float_as_uint(x) & 0xffffe000u), v = __uint_as_float(__float_as_uint(y) & 0xffffe000u);
  lead = half2_bits(__floats2half2_rn(u, v));
  float c = x - u, d = y - v;
  if constexpr (INFINITE) {
    c = fmaxf(c, fminf(x, 0x1p-24f));
    d = fmaxf(d, fminf(y, 0x1p-24f));
  }
  rest = half2_bits(__floats2half2_rn(c, d));
}

// Two pairs of stored bytes -> two f16 pairs.  i8: a byte u behind 0x64 is the half 1024 + u, less 1152 = u - 128.
// SEL: bytes (0, 1) and (2, 3) for K, whose pairs run along a row; (0, 2) and (1, 3) for V, whose transposed words
// hold two dimensions of two positions.
template <int F, bool V>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (F == kKvI8) {
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t x = __byte_perm(w, 0x64646464u, V ? 0x4240 : 0x4140);
    const uint32_t y = __byte_perm(w, 0x64646464u, V ? 0x4341 : 0x4342);
    a = half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&x), bias));
    b = half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&y), bias));
  } else {
    const uint32_t p = V ? __byte_perm(w, 0, 0x3120) : w;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(a), "=r"(b) : "r"(p));
  }
}

// Address of 16-byte piece c of row r of a K or V tile (boxes of kPart bytes a row, swizzled as the copy writes them).
template <int F, int HD, int KEYS>
__device__ __forceinline__ uint32_t piece(uint32_t base, int r, int c) {
  using Gm = Tile<F, HD, KEYS>;
  if constexpr (Gm::kPart == 128) return base + (c >> 3) * Gm::kBoxBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  else return base + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// The sequences: len[b] cached positions (clamped to the cache), and cum[b] units of one row tile and kv head before
// sequence b.
struct Seqs {
  const int32_t* cum;
  const int32_t* len;
};
struct SeqTables {
  int32_t cum[kMaxScan + 1], len[kMaxScan], sum[kMaxScan / 32];
};

__device__ __forceinline__ int units_of(int len, int unit, int lead) { return len ? (len + unit - 1) / unit + lead : 0; }

// Inclusive sums of the units of 32 sequences, one a lane.
__device__ __forceinline__ int scan32(int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, n, o);
    if (lane >= o) n += y;
  }
  return n;
}

// Every CTA makes the tables of up to kMaxScan sequences itself (larger batches: `given`, cum and then len); CTA 0 leaves
// the sums at `out` for the joining kernel.  For all threads of the CTA.
__device__ __forceinline__ Seqs sequences(const PrefixAttnArgs& a, const Plan& p, const int32_t* given, SeqTables& t, int32_t* out) {
  if (given) return Seqs{given, given + a.B + 1};
  if (p.own_nrt == 0) return Seqs{nullptr, nullptr};
  const int lane = threadIdx.x & 31, B = (int)a.B;
  for (int c = threadIdx.x >> 5; 32 * c < B; c += blockDim.x >> 5) {
    const int b = 32 * c + lane, len = b < B ? own_length(a, b, blockIdx.x == 0) : 0;
    const int n = scan32(b < B ? units_of(len, p.unit, p.lead) : 0);
    if (b < B) {
      t.len[b] = len;
      t.cum[b + 1] = n;
    }
    if (lane == 31) t.sum[c] = n;
  }
  __syncthreads();
  for (int c = threadIdx.x >> 5; 32 * c < B; c += blockDim.x >> 5) {
    int before = 0;
    for (int i = lane; i < c; i += 32) before += t.sum[i];
    before = __reduce_add_sync(0xffffffffu, before);
    const int b = 32 * c + lane;
    if (b < B) {
      const int n = t.cum[b + 1] + before;
      t.cum[b + 1] = n;
      if (blockIdx.x == 0) out[b + 1] = n;
    }
  }
  if (threadIdx.x == 0) {
    t.cum[0] = 0;
    if (blockIdx.x == 0) out[0] = 0;
  }
  __syncthreads();
  return Seqs{t.cum, t.len};
}

// ---------------------------------------------------------------- the walk over a worker's pieces

struct Piece {
  int64_t slot;      // item + worker
  int own;
  int z, kvh, rt;    // plane of the cache; kv head, row tile
  int seq;           // own items: the sequence
  int t0, t1;        // units of this worker
  int limit;         // positions that some row of the item sees
  int fewest;        // positions that every row sees
};

// The first unit of worker c: the first total % n workers take one unit more than the others.
__device__ __forceinline__ int share_start(int c, int total, int n, int each) {  // each = total / n
  return c * each + min(c, total - each * n);
}
// The worker that holds unit u < total.
__device__ __forceinline__ int share_of(int u, int total, int n, int each) {
  const int more = total - each * n, split = more * (each + 1);
  return u < split ? u / (each + 1) : more + (u - split) / each;
}

struct Walk {
  int u, end, b, worker;
  Walk() = default;
  __device__ Walk(const Plan& p, const PrefixAttnArgs& a, const Seqs& q, int worker_) : b(0), worker(worker_) {
    const int prefix = p.prefix_items * p.prefix_units, per = (int)a.own.heads * p.own_nrt;
    const int total = prefix + (per ? q.cum[a.B] * per : 0);
    const int each = total / p.by_workers;
    u = share_start(worker, total, p.workers, each);
    end = share_start(worker + 1, total, p.workers, each);
    if (end > prefix) {  // the last sequence whose units start at or before the first own unit
      const int first = max(u - prefix, 0);
      int lo = 0, hi = (int)a.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (q.cum[mid] * per <= first) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
    }
  }
  __device__ __forceinline__ bool next(Piece& x, const Plan& p, const PrefixAttnArgs& a, const Seqs& q) {
    while (u < end)
      if (step(x, p, a, q)) return true;
    return false;
  }
  // The next item's part; false if it has no keys.
  __device__ __forceinline__ bool step(Piece& x, const Plan& p, const PrefixAttnArgs& a, const Seqs& q) {
    const int prefix = p.prefix_items * p.prefix_units;
    int in, units;
    if (u >= prefix) {
      const int per = (int)a.own.heads * p.own_nrt, v = u - prefix;
      while (q.cum[b + 1] * per <= v) ++b;
      units = q.cum[b + 1] - q.cum[b];
      const int rest = v - q.cum[b] * per, j = rest / units;
      in = rest - j * units;
      x.slot = p.prefix_items + (int64_t)b * per + j;
      x.own = 1;
      x.kvh = j / p.by_own_nrt;
      x.rt = j - x.kvh * p.own_nrt;
      x.seq = b;
      x.z = b * (int)a.own.heads + x.kvh;
      const int first = x.rt * p.rt / p.by_G, last = (min((x.rt + 1) * p.rt, p.own_rows) - 1) / p.by_G;  // tokens
      const int seen = q.len[b] - (int)a.T + 1;
      x.limit = seen + last;
      x.fewest = seen + first;
    } else {
      units = p.prefix_units;
      x.slot = u / p.by_prefix_units;
      in = u - (int)x.slot * units;
      x.own = 0;
      x.kvh = (int)x.slot / p.by_prefix_nrt;
      x.rt = (int)x.slot - x.kvh * p.prefix_nrt;
      x.seq = 0;
      x.z = x.kvh;
      x.limit = x.fewest = (int)a.prefix_len;
    }
    const int n = min(units - in, end - u);
    x.t0 = max(0, in - p.lead);
    x.t1 = in + n - p.lead;
    x.slot += worker;
    u += n;
    return x.t1 > 0;
  }
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(umma::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// After a copy that was late: time for what is in flight to land before the shared memory is reused.
__device__ __noinline__ void grace() {
  const long long t0 = clock64();
  while (clock64() - t0 < 20000000LL) {}
}

// q row of logical row `row` of an item (null past the end) and the positions it sees.
template <typename Q>
__device__ __forceinline__ const Q* q_row(const PrefixAttnArgs& a, const Plan& p, const Piece& x, int row, int& lim) {
  const int rho = x.rt * p.rt + row;
  if (rho >= (x.own ? p.own_rows : p.prefix_rows)) {
    lim = 0;
    return nullptr;
  }
  const int b = x.own ? x.seq : rho / p.by_own_rows, in = x.own ? rho : rho - b * p.own_rows;
  const int t = in / p.by_G, g = in - t * p.G;
  lim = x.own ? x.fewest + t - x.rt * p.rt / p.by_G : x.limit;
  return static_cast<const Q*>(a.q) + (int64_t)b * a.qs.batch + t * a.qs.token + ((int64_t)x.kvh * p.G + g) * a.qs.head;
}

// A power of two that brings the largest of a folded row into [1, 2): its exponent leaves through the score factor, so
// that neither part of the split overflows or loses bits.  bits: max |q|; returns 2^-e.
__device__ __forceinline__ float row_shrink(uint32_t bits) {
  const uint32_t e = min(max(bits & 0x7f800000u, 64u << 23), 190u << 23);
  return __uint_as_float(0x7f000000u - e);
}

}  // namespace attn
}  // namespace uaii_b200
