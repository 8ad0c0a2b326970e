// prefix_attn.cu -- attention of new tokens over a prefix that the whole batch shares and each sequence's own
// cached positions, straight from an f16 or 8-bit cache (formats: kv_cache.cu).
//
//   s_j = scale * ks_j * (q . c_j),   out = sum_j e^(s_j - m) vs_j c'_j / sum_j e^(s_j - m)
//
// with c_j, c'_j the stored K and V values of position j and ks_j, vs_j their row scales (1 for f16).
// Token t of sequence b sees prefix positions [0, P) and own positions [0, own_len[b] - T + t]; a row that sees
// none is zero.  Running maximum, sums and outputs are f32.
//
// Work.  An item is a tile of query rows that read the same keys: (kv head, rows of the whole batch) over the
// prefix, (sequence, kv head, rows) over own positions.  Its keys come in tiles of 64; the tiles of all items, laid
// end to end, are dealt out evenly to the CTAs, so a CTA's share starts and ends inside items.  Every piece of an
// item leaves its unnormalised sums, row maxima and denominators in the workspace (slot = item + CTA, unique because
// each next piece raises one of the two), and a second kernel joins the pieces of each row in a fixed order.  Even
// CTAs take their share of the prefix first and odd ones their own positions: the first is bound by arithmetic, the
// second by memory, and an SM holds one of each.
//
// Products are warp-level f16 tensor-core MMAs with f32 accumulators.  Bytes become exact f16 operands in registers
// (the row scales act on scores and probabilities).  Two tilings of a 64-key tile over the four compute warps:
//   narrow  every warp takes the item's 8 or 16 rows and 16 of the keys (few rows: the keys are the work),
//   wide    every warp takes its own 32 operand rows and all keys (many rows: each key fragment feeds two MMAs).
// f32 queries are split in two f16 parts, and so are the probabilities: rows 0-7 of an MMA hold the leading parts and
// rows 8-15 the rests ("folded"), which keeps f32 accuracy at no cost while an item has no more than 8 rows.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cfloat>

#include "serve_kernels.hpp"
#include "umma.cuh"

namespace uaii_b200 {
namespace {

constexpr int kTile = 64;        // keys of a tile
constexpr int kWarps = 4;        // compute warps; one more warp copies
constexpr int kCtasPerSm = 2;
constexpr int kMaxGrid = 148 * kCtasPerSm;
constexpr int kMaxScan = 1024;   // sequences whose tile counts a CTA sums itself
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities carry a factor 2^14 (in sums and denominators alike): f16 then keeps 11 bits of every weight down to
// 2^-28 of the largest.
constexpr float kLift = 14.0f;

template <int F, int HD>
struct Geometry {
  static constexpr int kEsz = F == kKvF16 ? 2 : 1;
  static constexpr int kRow = HD * kEsz;                    // bytes of a stored row
  static constexpr int kPart = kRow < 128 ? kRow : 128;     // bytes of a row in one box (the swizzle span)
  static constexpr int kBoxes = kRow / kPart;
  static constexpr int kBoxBytes = kPart * kTile;
  static constexpr int kScaleBytes = F == kKvF16 ? 0 : 2 * kTile * 4;
  static constexpr int kStage = (2 * kBoxes * kBoxBytes + kScaleBytes + 1023) & ~1023;
  static constexpr int kStages = 70 * 1024 / kStage;        // what is in flight: two CTAs hold about 130 KB of an SM
  static constexpr int kShare = 32 * HD * 8;                // 128 operand rows of q, or the narrow tiling's merge
  static constexpr int kSmem = kStages * kStage + kShare + 1024;
};

struct Maps {
  CUtensorMap pk, pv, ok, ov;
};

struct Plan {
  int G;                 // query heads per kv head
  int prefix_rows;       // B * T * G
  int own_rows;          // T * G
  bool prefix_wide, own_wide;
  int prefix_rt, own_rt;          // rows of an item
  int prefix_nrt, own_nrt;        // items per kv head
  int64_t prefix_tiles;           // key tiles of a prefix item
  int64_t prefix_items;
  int grid;
  const int32_t* cum;    // tiles of the sequences before each [B + 1], or null: the CTAs sum them
  int32_t* cum_out;      // where CTA 0 leaves its sums for the joining kernel (null when cum is given)
  float* part;           // partial sums, prefix slots first
  float* ml;             // (maximum, denominator) of each partial row
  int64_t own_part0, own_ml0;     // offsets of the own slots
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
  asm volatile(
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
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

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
template <int F, int HD>
__device__ __forceinline__ uint32_t piece(uint32_t base, int r, int c) {
  using Gm = Geometry<F, HD>;
  if constexpr (Gm::kPart == 128) return base + (c >> 3) * Gm::kBoxBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  else return base + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// ---------------------------------------------------------------- one warp's running softmax

template <int F, int HD, bool FOLD, int MT>
struct Rows {
  static constexpr int kPer = FOLD ? 1 : 2;  // logical rows of a lane in one MMA tile
  float o[MT][HD / 8][4];
  float m[MT][kPer], l[MT][kPer];
  float f[MT][kPer];         // score factor: scale * log2(e), and the power of two taken out of a folded row of q
  int lim[MT][kPer];         // positions the row sees
  uint32_t vexp;             // exponent bits of the largest V scale so far (8-bit formats)

  // Leading part and rest.  Where an f16 cache holds an infinity, the rest is 0 * inf.
  static __device__ __forceinline__ float join(float lead, float rest) {
    if constexpr (F == kKvF16) return fabsf(lead) == INFINITY ? lead : lead + rest;
    return lead + rest;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][n][i] = 0.f;
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        m[t][r] = -INFINITY;
        l[t][r] = 0.f;
      }
    }
    vexp = 27u << 23;  // 2^-100
  }

  // Keys [key, key + 8 NT) of the tile at k_base / v_base, which starts at position pos0 and of
  // which some row sees the first `left`; masked says that some row may not see all of them.  a(ks, mt, frag) gives
  // the query operands.
  template <int NT, typename A>
  __device__ __forceinline__ void step(uint32_t k_base, uint32_t v_base, const float* ks, const float* vs, int key,
                                       int left, int pos0, bool masked, A&& a) {
    const int lane = threadIdx.x & 31, tq = lane & 3, mi = lane >> 3, r8 = lane & 7;
    float s[MT][NT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][n][i] = 0.f;
    // scores: four 16-byte pieces of eight keys at a time
    constexpr int kPieces = HD * Geometry<F, HD>::kEsz / 16;
#pragma unroll
    for (int c = 0; c < kPieces; c += 4) {
      constexpr int kSteps = F == kKvF16 ? 2 : 4;
      uint32_t q[kSteps][MT][4];
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) a((F == kKvF16 ? c / 2 : c) + j, t, q[j][t]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t w[4];
        ldsm4(w, piece<F, HD>(k_base, key + 8 * n + r8, c + mi));
        if constexpr (F == kKvF16) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma16816(s[t][n], q[0][t], w[0], w[1]);
            mma16816(s[t][n], q[1][t], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t b0, b1;
            unpack<F, false>(w[j], b0, b1);
#pragma unroll
            for (int t = 0; t < MT; ++t) mma16816(s[t][n], q[j][t], b0, b1);
          }
        }
      }
    }
    // columns 2 tq, 2 tq + 1 of each eight keys: K scales, and V scales as fractions of a power of two
    float kf[NT][2], vf[NT][2];
    float vshrink = 1.f;
    if constexpr (F != kKvF16) {
      uint32_t e = 0;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 x = *reinterpret_cast<const float2*>(ks + key + 8 * n + 2 * tq);
        const float2 y = *reinterpret_cast<const float2*>(vs + key + 8 * n + 2 * tq);
        kf[n][0] = x.x; kf[n][1] = x.y;
        vf[n][0] = y.x; vf[n][1] = y.y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (masked && key + 8 * n + 2 * tq + i >= left) vf[n][i] = 0.f;  // nothing is stored there
          const uint32_t b = __float_as_uint(vf[n][i]) & 0x7f800000u;
          e = max(e, b >= 254u << 23 ? 0u : b);  // a NaN scale shows in its products, not here
        }
      }
      e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
      e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
      if (e > vexp) {  // (the same in every lane)
        vshrink = __uint_as_float(max(0, (int)(0x3f800000u + vexp) - (int)e));
        vexp = e;
      }
      const float inv = __uint_as_float(0x7f000000u - vexp);  // its reciprocal
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        vf[n][0] *= inv;
        vf[n][1] *= inv;
      }
    }
    float off[MT][kPer];
    bool grew = vshrink != 1.f;
    float mn[MT][kPer];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        float mx = m[t][r];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float& x = s[t][n][2 * r + i];
            if constexpr (FOLD) x = join(x, s[t][n][2 + i]);
            if constexpr (F != kKvF16) x *= kf[n][i];
            if (!masked || pos0 + key + 8 * n + 2 * tq + i < lim[t][r]) mx = fmaxf(mx, x * f[t][r]);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mn[t][r] = mx;
        grew |= mx > m[t][r];
      }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
          const float c = mn[t][r] > m[t][r] ? ex2(m[t][r] - mn[t][r]) : 1.f, co = c * vshrink;
          m[t][r] = mn[t][r];
          l[t][r] *= c;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            o[t][n][2 * r] *= co;
            o[t][n][2 * r + 1] *= co;
            if constexpr (FOLD) {
              o[t][n][2] *= co;
              o[t][n][3] *= co;
            }
          }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < kPer; ++r) off[t][r] = kLift - (m[t][r] == -INFINITY ? 0.f : m[t][r]);
    // probabilities as operands, and their products with V: 16 keys at a time
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t p[MT][4];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < kPer; ++r) {
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool seen = !masked || pos0 + key + 8 * (n + h) + 2 * tq + i < lim[t][r];
              const float e = seen ? ex2(fmaf(s[t][n + h][2 * r + i], f[t][r], off[t][r])) : 0.f;
              l[t][r] += e;
              w[i] = e;
              if constexpr (F != kKvF16) w[i] = seen ? e * vf[n + h][i] : 0.f;
            }
            const __half2 lead = __floats2half2_rn(w[0], w[1]);
            p[t][2 * h + r] = half2_bits(lead);
            if constexpr (FOLD) {
              const float2 x = __half22float2(lead);
              p[t][2 * h + 1] = half2_bits(__floats2half2_rn(w[0] - x.x, w[1] - x.y));
            }
          }
#pragma unroll
      for (int c = 0; c < kPieces; c += 2) {
        uint32_t w[4];
        ldsm4t(w, piece<F, HD>(v_base, key + 8 * n + 8 * (mi & 1) + r8, c + (mi >> 1)));
        if constexpr (F == kKvF16) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma16816(o[t][c], p[t], w[0], w[1]);
            mma16816(o[t][c + 1], p[t], w[2], w[3]);
          }
        } else {  // a piece holds 16 dimensions: its even ones are tile 2 c, its odd ones tile 2 c + 1
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t e0, e1, d0, d1;
            unpack<F, true>(w[2 * j], e0, d0);
            unpack<F, true>(w[2 * j + 1], e1, d1);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              mma16816(o[t][2 * (c + j)], p[t], e0, e1);
              mma16816(o[t][2 * (c + j) + 1], p[t], d0, d1);
            }
          }
        }
      }
    }
  }

  // The row sums with V's power of two put back; l summed over the lanes of a row.
  __device__ __forceinline__ void finish() {
    const float up = F == kKvF16 ? 1.f : __uint_as_float(vexp);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        l[t][r] += __shfl_xor_sync(0xffffffffu, l[t][r], 1);
        l[t][r] += __shfl_xor_sync(0xffffffffu, l[t][r], 2);
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float& x = o[t][n][2 * r + i];
            if constexpr (FOLD) x = join(x, o[t][n][2 + i]);
            x *= up;
          }
      }
  }

  // Row r of tile t to dst[HD].
  __device__ __forceinline__ void store(float* dst, int t, int r) const {
    const int tq = threadIdx.x & 3;
    if constexpr (F == kKvF16) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
        *reinterpret_cast<float2*>(dst + 8 * n + 2 * tq) = make_float2(o[t][n][2 * r], o[t][n][2 * r + 1]);
    } else {
#pragma unroll
      for (int n = 0; n < HD / 8; n += 2)
        *reinterpret_cast<float4*>(dst + 8 * n + 4 * tq) =
            make_float4(o[t][n][2 * r], o[t][n + 1][2 * r], o[t][n][2 * r + 1], o[t][n + 1][2 * r + 1]);
    }
  }
};

// ---------------------------------------------------------------- the walk over a CTA's pieces

struct Piece {
  int64_t item;
  int64_t slot;      // item + CTA
  int kvh, rt;
  int64_t seq;       // own items: the sequence
  int t0, t1;        // key tiles of this CTA
  int limit;         // positions that some row of the item sees
};

// Walks the pieces of one CTA in one phase.
struct Walk {
  int64_t u, end;
  int64_t b = 0;     // own: the sequence of unit u
  bool own;
  const Plan& p;
  const PrefixAttnArgs& a;
  const int32_t* cum;
  __device__ Walk(const Plan& p_, const PrefixAttnArgs& a_, const int32_t* cum_, bool own_) : own(own_), p(p_), a(a_), cum(cum_) {
    const int64_t total = own ? (int64_t)cum[a.B] * a.own.heads * p.own_nrt : p.prefix_items * p.prefix_tiles;
    u = total * blockIdx.x / gridDim.x;
    end = total * (blockIdx.x + 1) / gridDim.x;
    if (own && u < end) {  // the last sequence whose units start at or before u
      const int64_t per = a.own.heads * p.own_nrt;
      int64_t lo = 0, hi = a.B - 1;
      while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (cum[mid] * per <= u) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
    }
  }
  __device__ bool next(Piece& x) {
    if (u >= end) return false;
    int64_t in, tiles;
    if (own) {
      const int64_t per = a.own.heads * p.own_nrt;
      while (cum[b + 1] * per <= u) ++b;
      tiles = cum[b + 1] - cum[b];
      const int64_t rest = u - cum[b] * per, j = rest / tiles;
      in = rest - j * tiles;
      x.item = b * per + j;
      x.kvh = (int)(j / p.own_nrt);
      x.rt = (int)(j % p.own_nrt);
      x.seq = b;
      const int last = min((x.rt + 1) * p.own_rt, p.own_rows) - 1;  // its token sees the most
      x.limit = own_length(a, b, false) - (int)a.T + last / p.G + 1;
    } else {
      tiles = p.prefix_tiles;
      x.item = u / tiles;
      in = u - x.item * tiles;
      x.kvh = (int)(x.item / p.prefix_nrt);
      x.rt = (int)(x.item % p.prefix_nrt);
      x.seq = 0;
      x.limit = (int)a.prefix_len;
    }
    const int64_t n = min(tiles - in, end - u);
    x.t0 = (int)in;
    // tiles that no row of the item sees are dealt out but not walked
    x.t1 = min((int)(in + n), max((int)in, (x.limit + kTile - 1) / kTile));
    x.slot = x.item + blockIdx.x;
    u += n;
    return true;
  }
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(umma::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  int stages;
  __device__ explicit Ring(int n) : stages(n) {}
  __device__ void advance() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

template <int STAGES>
struct Control {
  uint64_t full[STAGES], empty[STAGES];
  int abort;
  float ml[kWarps][16][2];
  int32_t cum[kMaxScan + 1];
};

// q row of logical row `row` of an item (null past the end) and the positions it sees.
template <typename Q>
__device__ __forceinline__ const Q* q_row(const PrefixAttnArgs& a, const Plan& p, const Piece& x, bool own, int row, int& lim) {
  const int rho = x.rt * (own ? p.own_rt : p.prefix_rt) + row;
  if (rho >= (own ? p.own_rows : p.prefix_rows)) {
    lim = 0;
    return nullptr;
  }
  const int64_t b = own ? x.seq : rho / p.own_rows;
  const int in = own ? rho : rho % p.own_rows;
  const int t = in / p.G, g = in % p.G;
  lim = own ? x.limit - (min((x.rt + 1) * p.own_rt, p.own_rows) - 1) / p.G + t : x.limit;
  return static_cast<const Q*>(a.q) + b * a.qs.batch + t * a.qs.token + ((int64_t)x.kvh * p.G + g) * a.qs.head;
}

// A power of two that brings the largest of a folded row into [1, 2): its exponent leaves through the score factor, so
// that neither part of the split overflows or loses bits.  bits: max |q|; returns 2^-e.
__device__ __forceinline__ float row_shrink(uint32_t bits) {
  const uint32_t e = min(max(bits & 0x7f800000u, 64u << 23), 190u << 23);
  return __uint_as_float(0x7f000000u - e);
}

// Rows of the last tile past the end of the cached positions hold other data: V of f16 and e4m3 may be NaN there.
template <int F, int HD>
__device__ __forceinline__ void zero_v(uint8_t* v, int from, int to, int thread, int threads) {
  using Gm = Geometry<F, HD>;
  constexpr int kPer = Gm::kPart / 16;
  for (int i = thread; i < (to - from) * kPer * Gm::kBoxes; i += threads) {
    const int box = i / ((to - from) * kPer), j = i % ((to - from) * kPer);
    *reinterpret_cast<uint4*>(v + box * Gm::kBoxBytes + (from + j / kPer) * Gm::kPart + (j % kPer) * 16) = make_uint4(0, 0, 0, 0);
  }
  umma::fence_proxy_async_smem();
}

template <int F, int HD, bool FOLD, bool WIDE, typename Q, typename C>
__device__ void consume(const PrefixAttnArgs& a, const Plan& p, Walk w, bool own, uint8_t* smem, C& ctl, Ring& ring) {
  using Gm = Geometry<F, HD>;
  constexpr int MT = WIDE ? 2 : 1;
  constexpr int RPT = FOLD ? 8 : 16;                       // logical rows of an MMA tile
  constexpr int RT = (WIDE ? kWarps * MT : 1) * RPT;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, tq = lane & 3;
  uint8_t* share = smem + Gm::kStages * Gm::kStage;
  Rows<F, HD, FOLD, MT> st;
  const float base = a.scale * kLog2e;
  Piece x;
  while (w.next(x)) {
    st.clear();
    uint32_t qa[WIDE ? 1 : HD / 16][4];
    if constexpr (WIDE) {
      // 128 operand rows of q in shared memory, 16-byte pieces swizzled, one thread a row
      const int tile = t >> 4, r = t & 15;                  // operand row t: MMA tile t / 16
      const int row = tile * RPT + (FOLD ? r & 7 : r);
      int lim;
      const Q* src = q_row<Q>(a, p, x, own, row, lim);
      float shrink = 1.f;
      if constexpr (FOLD) {
        uint32_t mx = 0;
        if (src)
          for (int d = 0; d < HD; ++d) mx = max(mx, __float_as_uint((float)src[d]) & 0x7fffffffu);
        shrink = row_shrink(mx);
      }
      for (int c = 0; c < HD / 8; ++c) {  // the eight operand positions of piece c
        __half h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          int d = 8 * c + i;                                 // operand position -> dimension
          if constexpr (F != kKvF16) d = (d & ~15) | ((d & 6) << 1) | ((d & 8) >> 2) | (d & 1);
          const float y = src ? (float)src[d] * shrink : 0.f;
          const __half lead = __float2half_rn(y);
          h[i] = FOLD && (r & 8) ? __float2half_rn(y - __half2float(lead)) : lead;
        }
        *reinterpret_cast<uint4*>(share + t * (2 * HD) + ((c ^ (t & 7)) << 4)) = *reinterpret_cast<const uint4*>(h);
      }
      if constexpr (FOLD) {
        if (!(r & 8)) ctl.ml[warp][(tile & 1) * 8 + (r & 7)][0] = 1.f / shrink;
      }
      compute_barrier();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r2 = 0; r2 < (FOLD ? 1 : 2); ++r2) {
          (void)q_row<Q>(a, p, x, own, (warp * MT + m) * RPT + g + 8 * r2, st.lim[m][r2]);
          st.f[m][r2] = FOLD ? base * ctl.ml[warp][m * 8 + g][0] : base;
        }
    } else {
      const Q* src[2];
#pragma unroll
      for (int r = 0; r < (FOLD ? 1 : 2); ++r) {
        src[r] = q_row<Q>(a, p, x, own, g + 8 * r, st.lim[0][r]);
        st.f[0][r] = base;
      }
      float shrink = 1.f;
      if constexpr (FOLD && sizeof(Q) == 4) {
        uint32_t mx = 0;
        if (src[0])
          for (int d = tq; d < HD; d += 4) mx = max(mx, __float_as_uint((float)src[0][d]) & 0x7fffffffu);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        shrink = row_shrink(mx);
        st.f[0][0] = base / shrink;
      }
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // elements 2 tq, 2 tq + 1 (+ 8)
          const int d = F == kKvF16 ? 16 * ks + 8 * h + 2 * tq : 16 * ks + 4 * tq + 2 * h;
#pragma unroll
          for (int r = 0; r < (FOLD ? 1 : 2); ++r) {
            const float y0 = src[r] ? (float)src[r][d] * shrink : 0.f, y1 = src[r] ? (float)src[r][d + 1] * shrink : 0.f;
            const __half2 lead = __floats2half2_rn(y0, y1);
            qa[ks][2 * h + r] = half2_bits(lead);
            if constexpr (FOLD) {
              const float2 z = __half22float2(lead);
              qa[ks][2 * h + 1] = half2_bits(__floats2half2_rn(y0 - z.x, y1 - z.y));
            }
          }
        }
    }
    for (int kt = x.t0; kt < x.t1; ++kt) {
      umma::bounded_wait(&ctl.full[ring.stage], ring.phase, &ctl.abort, a.err, kErrKvCopy);
      uint8_t* stage = smem + ring.stage * Gm::kStage;
      const uint32_t k_base = umma::smem_u32(stage), v_base = k_base + Gm::kBoxes * Gm::kBoxBytes;
      const float* ks = reinterpret_cast<const float*>(stage + 2 * Gm::kBoxes * Gm::kBoxBytes);
      const int pos0 = kt * kTile, left = x.limit - pos0;
      // every row of a prefix item sees the same positions; the first row of an own item sees the fewest
      const int fewest = own ? x.limit - (min((x.rt + 1) * p.own_rt, p.own_rows) - 1) / p.G + x.rt * p.own_rt / p.G : x.limit;
      const bool masked = pos0 + kTile > fewest;
      if (F != kKvI8 && left < kTile) {
        uint8_t* v = stage + Gm::kBoxes * Gm::kBoxBytes;
        if constexpr (WIDE) {
          zero_v<F, HD>(v, left, kTile, t, 32 * kWarps);
          compute_barrier();
        } else {
          if (left < 16 * warp + 16) zero_v<F, HD>(v, max(left, 16 * warp), 16 * warp + 16, lane, 32);
          __syncwarp();
        }
      }
      if constexpr (WIDE) {
        auto frag = [&](int step, int m, uint32_t (&f)[4]) {
          // matrices: rows 0-7 and 8-15 of the tile, pieces 2 step and 2 step + 1
          const int row = (warp * MT + m) * 16 + (lane & 15), c = 2 * step + (lane >> 4);
          ldsm4(f, umma::smem_u32(share) + row * (2 * HD) + ((c ^ (row & 7)) << 4));
        };
#pragma unroll 1
        for (int key = 0; key < kTile; key += 32)
          st.template step<4>(k_base, v_base, ks, ks + kTile, key, left, pos0, masked, frag);
      } else {
        st.template step<2>(k_base, v_base, ks, ks + kTile, 16 * warp, left, pos0, masked, [&](int step, int, uint32_t (&f)[4]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = qa[step][i];
        });
      }
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(&ctl.empty[ring.stage]);
      ring.advance();
    }
    if constexpr (WIDE) compute_barrier();  // q's rows and scales are free again
    st.finish();
    const int64_t rows = x.slot * RT;
    float* part = p.part + (own ? p.own_part0 : 0) + rows * HD;
    float* ml = p.ml + (own ? p.own_ml0 : 0) + rows * 2;
    if constexpr (WIDE) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < (FOLD ? 1 : 2); ++r) {
          const int row = (warp * MT + m) * RPT + g + 8 * r;
          st.store(part + (int64_t)row * HD, m, r);
          if (tq == 0) *reinterpret_cast<float2*>(ml + 2 * row) = make_float2(st.m[m][r], st.l[m][r]);
        }
    } else {
      // join the four warps' keys
      float* mine = reinterpret_cast<float*>(share) + warp * RT * HD;
#pragma unroll
      for (int r = 0; r < (FOLD ? 1 : 2); ++r) {
        st.store(mine + (g + 8 * r) * HD, 0, r);
        if (tq == 0) {
          ctl.ml[warp][g + 8 * r][0] = st.m[0][r];
          ctl.ml[warp][g + 8 * r][1] = st.l[0][r];
        }
      }
      compute_barrier();
      for (int i = t; i < RT * HD / 4; i += 32 * kWarps) {
        const int row = i / (HD / 4);
        float mx = ctl.ml[0][row][0];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) mx = fmaxf(mx, ctl.ml[k][row][0]);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float f = mx == -INFINITY ? 1.f : ex2(ctl.ml[k][row][0] - mx);
          const float4 y = reinterpret_cast<const float4*>(share)[k * (RT * HD / 4) + i];
          s.x = fmaf(f, y.x, s.x);
          s.y = fmaf(f, y.y, s.y);
          s.z = fmaf(f, y.z, s.z);
          s.w = fmaf(f, y.w, s.w);
          l = fmaf(f, ctl.ml[k][row][1], l);
        }
        reinterpret_cast<float4*>(part)[i] = s;
        if (i % (HD / 4) == 0) *reinterpret_cast<float2*>(ml + 2 * row) = make_float2(mx, l);
      }
      compute_barrier();
    }
  }
}

template <int F, int HD, typename C>
__device__ void produce(const PrefixAttnArgs& a, const Maps& maps, Walk w, bool own, uint8_t* smem, C& ctl, Ring& ring) {
  using Gm = Geometry<F, HD>;
  const int lane = threadIdx.x & 31;
  const KvCache& c = own ? a.own : a.prefix;
  const CUtensorMap *mk = own ? &maps.ok : &maps.pk, *mv = own ? &maps.ov : &maps.pv;
  Piece x;
  while (w.next(x)) {
    const int z = (int)(own ? x.seq * a.own.heads + x.kvh : x.kvh);
    for (int kt = x.t0; kt < x.t1; ++kt) {
      const bool ok = umma::bounded_wait(&ctl.empty[ring.stage], ring.phase ^ 1, &ctl.abort, a.err, kErrKvCopy);
      if (!ok) return;
      uint8_t* stage = smem + ring.stage * Gm::kStage;
      uint64_t* bar = &ctl.full[ring.stage];
      if (lane == 0) {
        umma::mbar_arrive_expect_tx(bar, 2 * Gm::kBoxes * Gm::kBoxBytes);
        const uint32_t dst = umma::smem_u32(stage);
#pragma unroll
        for (int b = 0; b < Gm::kBoxes; ++b) {
          tma_load_3d(dst + b * Gm::kBoxBytes, mk, bar, b * (Gm::kPart / Gm::kEsz), kt * kTile, z);
          tma_load_3d(dst + (Gm::kBoxes + b) * Gm::kBoxBytes, mv, bar, b * (Gm::kPart / Gm::kEsz), kt * kTile, z);
        }
      }
      if constexpr (F != kKvF16) {  // row scales: 4-byte copies, zero past the end of the cache
        const uint32_t dst = umma::smem_u32(stage + 2 * Gm::kBoxes * Gm::kBoxBytes);
#pragma unroll
        for (int i = 0; i < 2 * kTile / 32; ++i) {
          const int j = (i % (kTile / 32)) * 32 + lane;
          const int64_t pos = (int64_t)kt * kTile + j;
          const bool in = pos < c.max_seq;
          const float* src = (i < kTile / 32 ? c.k_scale : c.v_scale) + (int64_t)z * c.max_seq + (in ? pos : 0);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + (i * 32 + lane) * 4), "l"(src), "r"(in ? 4 : 0)
                       : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(umma::smem_u32(bar)) : "memory");
      }
      __syncwarp();
      ring.advance();
    }
  }
}

template <int F, int HD, typename Q, bool NARROW_FOLD>
__global__ void __launch_bounds__(32 * (kWarps + 1), kCtasPerSm)
    prefix_attn_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan p, const __grid_constant__ Maps maps) {
  using Gm = Geometry<F, HD>;
  constexpr bool kFold = sizeof(Q) == 4;  // the wide tiling splits f32 queries
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ Control<Gm::kStages> ctl;
  const int t = threadIdx.x;
  if (t == 0) {
    for (int i = 0; i < Gm::kStages; ++i) {
      umma::mbar_init(&ctl.full[i], F == kKvF16 ? 1 : 33);
      umma::mbar_init(&ctl.empty[i], kWarps);
    }
    ctl.abort = 0;
    umma::fence_barrier_init();
  }
  const int32_t* cum = p.cum;
  if (cum == nullptr) {  // key tiles of the sequences before each
    const int lane = t & 31;
    if (t < 32) {
      int sum = 0;
      for (int b0 = 0; b0 < (int)a.B; b0 += 32) {
        const int b = b0 + lane;
        int n = b < a.B ? (own_length(a, b, blockIdx.x == 0) + kTile - 1) / kTile : 0;
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, n, o);
          if (lane >= o) n += y;
        }
        if (b < a.B) ctl.cum[b + 1] = sum + n;
        sum += __shfl_sync(0xffffffffu, n, 31);
      }
      if (lane == 0) ctl.cum[0] = 0;
    }
    cum = ctl.cum;
  }
  __syncthreads();
  if (p.cum == nullptr && blockIdx.x == 0)
    for (int i = t; i <= a.B; i += blockDim.x) p.cum_out[i] = ctl.cum[i];
  Ring ring(Gm::kStages);
  for (int i = 0; i < 2; ++i) {
    const bool own = (i ^ (blockIdx.x & 1)) != 0;
    if (!own && p.prefix_items == 0) continue;
    Walk w(p, a, cum, own);
    if (t >= 32 * kWarps) produce<F, HD>(a, maps, w, own, smem, ctl, ring);
    else if (own ? p.own_wide : p.prefix_wide) consume<F, HD, kFold, true, Q>(a, p, w, own, smem, ctl, ring);
    else consume<F, HD, NARROW_FOLD, false, Q>(a, p, w, own, smem, ctl, ring);
  }
  if (*(volatile int*)&ctl.abort) {  // a copy was late: give what is in flight time to land before the memory is reused
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000LL) {}
  }
}

// Key tiles of the sequences before each, for batches too large for a CTA's shared memory.
__global__ void __launch_bounds__(1024) tile_sums_kernel(const __grid_constant__ PrefixAttnArgs a, int32_t* cum) {
  __shared__ int warp_sum[32];
  const int t = threadIdx.x, lane = t & 31;
  int before = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += 1024) {
    const int64_t b = b0 + t;
    int n = b < a.B ? (own_length(a, b, true) + kTile - 1) / kTile : 0;
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += y;
    }
    if (lane == 31) warp_sum[t >> 5] = n;
    __syncthreads();
    int all = 0;
    for (int i = 0; i < 32; ++i) {
      if (i == (t >> 5)) n += all;
      all += warp_sum[i];
    }
    if (b < a.B) cum[b + 1] = before + n;
    before += all;
    __syncthreads();
  }
  if (t == 0) cum[0] = 0;
}

// out = sum over a row's pieces of 2^(m - M) o / sum of 2^(m - M) l, prefix pieces first.  One warp per row.
template <int HD, typename Q>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan p,
                                                   const int32_t* __restrict__ cum) {
  constexpr int N = HD / 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= a.B * a.T * a.H) return;
  const int64_t h = row % a.H, bt = row / a.H, b = bt / a.T, t = bt % a.T;
  const int64_t kvh = h / p.G, g = h % p.G;
  float mx = -INFINITY, l = 0.f, o[N] = {};
  for (int own = p.prefix_items ? 0 : 1; own < 2; ++own) {
    const int64_t rho = own ? t * p.G + g : (b * a.T + t) * p.G + g;
    const int rt = own ? p.own_rt : p.prefix_rt;
    const int64_t j = rho / rt, in = rho % rt;
    int64_t item, u0, tiles, total;
    if (own) {
      const int64_t per = a.own.heads * p.own_nrt;
      tiles = cum[b + 1] - cum[b];
      item = b * per + kvh * p.own_nrt + j;
      u0 = cum[b] * per + (kvh * p.own_nrt + j) * tiles;
      total = cum[a.B] * per;
    } else {
      tiles = p.prefix_tiles;
      item = kvh * p.prefix_nrt + j;
      u0 = item * tiles;
      total = p.prefix_items * tiles;
    }
    if (tiles == 0) continue;
    // CTA c holds units [total c / grid, total (c + 1) / grid)
    int64_t c = u0 * p.grid / total;
    while (total * (c + 1) / p.grid <= u0) ++c;
    for (; c < p.grid && total * c / p.grid < u0 + tiles; ++c) {
      if (total * c / p.grid == total * (c + 1) / p.grid) continue;  // an idle CTA
      const int64_t r = (item + c) * rt + in;
      const float2 ml = *reinterpret_cast<const float2*>(p.ml + (own ? p.own_ml0 : 0) + 2 * r);
      const float* src = p.part + (own ? p.own_part0 : 0) + r * HD + N * lane;
      const float mn = fmaxf(mx, ml.x), safe = mn == -INFINITY ? 0.f : mn;
      const float fo = ex2(mx - safe), fn = ex2(ml.x - safe);
      mx = mn;
      l = l * fo + ml.y * fn;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = o[i] * fo + src[i] * fn;
    }
  }
  Q* out = static_cast<Q*>(a.out) + row * HD + N * lane;
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (Q)(l == 0.f ? 0.f : __fdiv_rn(o[i], l));
}

// ---------------------------------------------------------------- host side

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr{};
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr);
    return e == cudaSuccess && qr == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
  }();
  return fn;
}

// [batch * heads, max_seq, hd] as boxes of 64 positions of at most 128 bytes; positions past max_seq read as zero.
bool make_map(CUtensorMap* map, const KvCache& c, const void* data) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t esz = c.fmt == kKvF16 ? 2 : 1, row = esz * c.hd;
  const cuuint32_t span = (cuuint32_t)(row < 128 ? row : 128);
  const cuuint64_t dims[3] = {(cuuint64_t)c.hd, (cuuint64_t)c.max_seq, (cuuint64_t)(c.batch * c.heads)};
  const cuuint64_t strides[2] = {row, row * (cuuint64_t)c.max_seq};
  const cuuint32_t box[3] = {(cuuint32_t)(span / esz), (cuuint32_t)kTile, 1}, es[3] = {1, 1, 1};
  return enc(map, c.fmt == kKvF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
             const_cast<void*>(data), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct Layout {
  Plan p;
  int64_t prefix_slots, own_slots;
  size_t part, ml, bytes;
};

Layout lay_out(const PrefixAttnArgs& a) {
  Layout l{};
  Plan& p = l.p;
  p.G = (int)(a.H / a.own.heads);
  p.own_rows = (int)(a.T * p.G);
  p.prefix_rows = (int)(a.B * p.own_rows);
  const int wide = a.half ? 128 : 64;
  const auto tile_of = [&](int rows, bool* w) {
    *w = rows > 16;
    return *w ? wide : a.half && rows > 8 ? 16 : 8;
  };
  p.own_rt = tile_of(p.own_rows, &p.own_wide);
  p.prefix_rt = tile_of(p.prefix_rows, &p.prefix_wide);
  // one narrow tiling per launch: 16 rows of f16 when either side has more than 8
  if (a.half && a.prefix_len && !p.own_wide && !p.prefix_wide && p.own_rt != p.prefix_rt) p.own_rt = p.prefix_rt = 16;
  p.own_nrt = (p.own_rows + p.own_rt - 1) / p.own_rt;
  p.prefix_nrt = (p.prefix_rows + p.prefix_rt - 1) / p.prefix_rt;
  p.prefix_tiles = (a.prefix_len + kTile - 1) / kTile;
  p.prefix_items = a.prefix_len ? a.own.heads * p.prefix_nrt : 0;
  const int64_t own_items = a.B * a.own.heads * p.own_nrt;
  const int64_t most = p.prefix_items * p.prefix_tiles + own_items * ((a.own.max_seq + kTile - 1) / kTile);
  p.grid = (int)(most < kMaxGrid ? most : kMaxGrid);
  l.prefix_slots = p.prefix_items ? p.prefix_items + p.grid : 0;
  l.own_slots = own_items + p.grid;
  const int64_t prefix_rows = l.prefix_slots * p.prefix_rt, rows = prefix_rows + l.own_slots * p.own_rt;
  p.own_part0 = prefix_rows * a.own.hd;
  p.own_ml0 = prefix_rows * 2;
  l.part = up256(sizeof(int32_t) * (size_t)(a.B + 1));
  l.ml = l.part + up256(sizeof(float) * (size_t)(rows * a.own.hd));
  l.bytes = l.ml + up256(sizeof(float) * (size_t)(rows * 2));
  return l;
}

template <int F, int HD, typename Q, bool NARROW_FOLD>
cudaError_t run(const PrefixAttnArgs& a, const Plan& p, const Maps& maps, cudaStream_t st) {
  const auto kern = prefix_attn_kernel<F, HD, Q, NARROW_FOLD>;
  constexpr int smem = Geometry<F, HD>::kSmem;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)p.grid, 32 * (kWarps + 1), smem, st>>>(a, p, maps);
  return cudaGetLastError();
}

template <int F, int HD>
cudaError_t run_type(const PrefixAttnArgs& a, const Plan& p, const Maps& maps, cudaStream_t st) {
  if (!a.half) return run<F, HD, float, true>(a, p, maps, st);
  const bool sixteen = (!p.own_wide && p.own_rt == 16) || (!p.prefix_wide && p.prefix_items && p.prefix_rt == 16);
  return sixteen ? run<F, HD, __half, false>(a, p, maps, st) : run<F, HD, __half, true>(a, p, maps, st);
}

template <int F>
cudaError_t run_dim(const PrefixAttnArgs& a, const Plan& p, const Maps& maps, cudaStream_t st) {
  return a.own.hd == 128 ? run_type<F, 128>(a, p, maps, st) : run_type<F, 64>(a, p, maps, st);
}

}  // namespace

size_t prefix_attn_ws(const PrefixAttnArgs& a) { return lay_out(a).bytes; }

cudaError_t launch_prefix_attn(const PrefixAttnArgs& a, void* ws, int* launches, cudaStream_t st) {
  Layout l = lay_out(a);
  Plan& p = l.p;
  char* base = static_cast<char*>(ws);
  int32_t* cum = reinterpret_cast<int32_t*>(base);
  p.part = reinterpret_cast<float*>(base + l.part);
  p.ml = reinterpret_cast<float*>(base + l.ml);
  Maps maps;
  if (!make_map(&maps.ok, a.own, a.own.k) || !make_map(&maps.ov, a.own, a.own.v)) return cudaErrorInvalidValue;
  if (p.prefix_items && (!make_map(&maps.pk, a.prefix, a.prefix.k) || !make_map(&maps.pv, a.prefix, a.prefix.v)))
    return cudaErrorInvalidValue;
  *launches = 2;
  if (a.B > kMaxScan) {
    tile_sums_kernel<<<1, 1024, 0, st>>>(a, cum);
    p.cum = cum;
    *launches = 3;
  } else {
    p.cum_out = cum;
  }
  cudaError_t e = a.own.fmt == kKvI8     ? run_dim<kKvI8>(a, p, maps, st)
                  : a.own.fmt == kKvE4M3 ? run_dim<kKvE4M3>(a, p, maps, st)
                                         : run_dim<kKvF16>(a, p, maps, st);
  if (e != cudaSuccess) return e;
  const unsigned blocks = (unsigned)((a.B * a.T * a.H + 3) / 4);
  if (a.half) {
    if (a.own.hd == 128) join_kernel<128, __half><<<blocks, 128, 0, st>>>(a, p, cum);
    else join_kernel<64, __half><<<blocks, 128, 0, st>>>(a, p, cum);
  } else {
    if (a.own.hd == 128) join_kernel<128, float><<<blocks, 128, 0, st>>>(a, p, cum);
    else join_kernel<64, float><<<blocks, 128, 0, st>>>(a, p, cum);
  }
  return cudaGetLastError();
}

}  // namespace uaii_b200
