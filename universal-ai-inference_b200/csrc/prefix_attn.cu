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
// prefix, (sequence, kv head, rows) over own positions.  Its keys come in units; the units of all items, laid end to
// end, are dealt out evenly to the CTAs, so a CTA's share starts and ends inside items.  Every piece of an item leaves
// its unnormalised sums, row maxima and denominators in the workspace (slot = item + CTA, unique because each next
// piece raises one of the two), and a last kernel joins the pieces of each row in a fixed order.
//
// Two tilings, one kernel each.  Bytes become exact f16 operands (the row scales act on scores and probabilities);
// accumulators are f32.
//   narrow  8 or 16 rows; every warp takes other keys of the piece, from copies of its own (few rows: the keys are
//           the work, and the kernel is bound by the cache's bytes).
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

constexpr int kSms = 148;
constexpr int kTile = 64;        // wide: keys of a tile
constexpr int kWarps = 4;        // compute warps (wide: one more warp copies)
constexpr int kWideCtas = 2, kNarrowCtas = 3;  // per SM
constexpr int kMaxScan = 1024;   // sequences whose tile counts a CTA sums itself
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are 2^(s - m + 8) (in sums and denominators alike), and m follows the running maximum only when that
// rises by more than 6: the sums are then seldom rescaled, weights stay below 2^14 (2^15 with V's scale, a fraction
// below 2), and f16 keeps 11 bits of each down to 2^-22 of the largest.
constexpr float kLift = 8.0f, kSlack = 6.0f;

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

template <int F, int HD>
struct Wide {
  using Tl = Tile<F, HD, kTile>;
  static constexpr int kStage = (2 * Tl::kBytes + Tl::kScaleBytes + 1023) & ~1023;
  static constexpr int kStages = 70 * 1024 / kStage;        // in flight: two CTAs hold about 130 KB of an SM
  static constexpr int kShare = 32 * HD * 8;                // 128 operand rows of q
  static constexpr int kSmem = kStages * kStage + kShare + 1024;
};

// Narrow: each warp copies for itself, kKeys positions at a time, the next ones while it works.  Three CTAs of four
// warps hold 190 KB of an SM, about half of it in flight.
template <int F, int HD>
struct Narrow {
  static constexpr int kKeys = F == kKvF16 && HD == 128 ? 16 : 32;
  using Tl = Tile<F, HD, kKeys>;
  static constexpr int kStage = 2 * Tl::kBytes;             // 4, 8 or (f16 of 16 keys) 8 KB
  static constexpr int kStages = 16 * 1024 / kStage;
  static constexpr int kScales = kStages * Tl::kScaleBytes; // of one warp, after all the tiles
  static constexpr int kSmem = kWarps * (kStages * kStage + kScales) + 1024;
  static constexpr int kUnit = kWarps * kKeys;
};

struct Maps {
  CUtensorMap pk, pv, ok, ov;
};

// The items of one kernel: prefix items first, then own ones (either may be missing).
struct Plan {
  int G;                   // query heads per kv head
  int prefix_rows;         // B * T * G
  int own_rows;            // T * G
  int rt;                  // rows of an item
  int unit;                // keys of a unit
  int prefix_nrt, own_nrt; // items per kv head (0: none)
  int prefix_units;        // units of a prefix item
  int prefix_items;
  int grid;                // CTAs (0: the kernel has no work)
  float* part;             // partial sums [slot][rt][hd]
  float* ml;               // (maximum, denominator) of each partial row
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
template <int F, int HD, int KEYS>
__device__ __forceinline__ uint32_t piece(uint32_t base, int r, int c) {
  using Gm = Tile<F, HD, KEYS>;
  if constexpr (Gm::kPart == 128) return base + (c >> 3) * Gm::kBoxBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  else return base + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// ---------------------------------------------------------------- one warp's running softmax

template <int F, int HD, bool FOLD, int MT, int KEYS>
struct Rows {
  static constexpr int kPer = FOLD ? 1 : 2;  // logical rows of a lane in one MMA tile
  static constexpr int kPieces = HD * Tile<F, HD, KEYS>::kEsz / 16;  // 16-byte pieces of a row
  // The two parts of a weight resolve 2^-24, f16's smallest step.  Smaller weights are added in passes of their own,
  // 20 binary orders at a time, raised to [2^-6, 2^14): only very uneven scores (22 e-foldings) need them.
  static constexpr bool kFar = FOLD && MT == 1;
  static constexpr float kNear = -24.f;
  float o[MT][HD / 8][4];
  float m[MT][kPer], l[MT][kPer];
  float f[MT][kPer];         // score factor: scale * log2(e), and the power of two taken out of a folded row of q
  int lim[MT][kPer];         // positions the row sees
  float vtop;                // a power of two above every V scale so far (8-bit formats)

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
    vtop = 0x1p-100f;
  }

  // Keys [key, key + 8 NT) of the tile at k_base / v_base, which starts at position pos0 and of
  // which some row sees the first `left`; masked says that some row may not see all of them.  a(ks, mt, frag) gives
  // the query operands.
  template <int NT, bool masked, typename A>
  __device__ __forceinline__ void step(uint32_t k_base, uint32_t v_base, const float* ks, const float* vs, int key,
                                       int left, int pos0, A&& a) {
    const int lane = threadIdx.x & 31, tq = lane & 3, mi = lane >> 3, r8 = lane & 7;
    float s[MT][NT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][n][i] = 0.f;
    // scores: four 16-byte pieces of eight keys at a time
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
        ldsm4(w, piece<F, HD, KEYS>(k_base, key + 8 * n + r8, c + mi));
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
    if constexpr (F != kKvF16) {
      float most = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 x = *reinterpret_cast<const float2*>(ks + key + 8 * n + 2 * tq);
        const float2 y = *reinterpret_cast<const float2*>(vs + key + 8 * n + 2 * tq);
        kf[n][0] = x.x; kf[n][1] = x.y;
        vf[n][0] = y.x; vf[n][1] = y.y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (masked && key + 8 * n + 2 * tq + i >= left) vf[n][i] = 0.f;  // nothing is stored there
          most = fmaxf(most, vf[n][i]);                                    // (a NaN shows in its products, not here)
        }
      }
      if (__any_sync(0xffffffffu, most >= vtop)) raise_v(most);
      const float inv = __uint_as_float(0x7f800000u - __float_as_uint(vtop));  // 2 / vtop
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        vf[n][0] *= inv;
        vf[n][1] *= inv;
      }
    }
    // exponents against the reference; a lane checks its own, the row's maximum is only made when one is too large
    bool grew = false;
    float x[MT][kPer][NT][2];
    auto exponents = [&]() {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
          const float off = kLift - (m[t][r] == -INFINITY ? 0.f : m[t][r]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              x[t][r][n][i] = fmaf(s[t][n][2 * r + i], F == kKvF16 ? f[t][r] : kf[n][i] * f[t][r], off);
        }
    };
    auto seen = [&](int t, int r, int n, int i) { return !masked || pos0 + key + 8 * n + 2 * tq + i < lim[t][r]; };
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if constexpr (FOLD) s[t][n][i] = join(s[t][n][i], s[t][n][2 + i]);
    exponents();
    float mx[MT][kPer];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        mx[t][r] = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (seen(t, r, n, i)) mx[t][r] = fmaxf(mx[t][r], x[t][r][n][i]);
        grew |= mx[t][r] > (m[t][r] == -INFINITY ? -INFINITY : kLift + kSlack);
      }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
          float y = mx[t][r];
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
          y += (m[t][r] == -INFINITY ? 0.f : m[t][r]) - kLift;
          // whole numbers, so that neither the factors nor the differences to them round
          const float to = fmaxf(m[t][r], ceilf(y));
          const float c = to > m[t][r] ? ex2(m[t][r] - to) : 1.f;
          m[t][r] = to;
          l[t][r] *= c;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            o[t][n][2 * r] *= c;
            o[t][n][2 * r + 1] *= c;
            if constexpr (FOLD) {
              o[t][n][2] *= c;
              o[t][n][3] *= c;
            }
          }
        }
      exponents();
    }
    float low = 0.f;  // the smallest exponent
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < kPer; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (kFar && seen(t, r, n, i)) low = fminf(low, x[t][r][n][i]);
    const bool far = kFar && __any_sync(0xffffffffu, low < kNear);
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t p[MT][4];
      weigh(x, vf, n, seen, [&](int t, int r, float y, float e) {
        l[t][r] += e;
        return far && y < kNear ? 0.f : e;
      }, p);
      products(v_base, key + 8 * n, [&](int c, int t, uint32_t b0, uint32_t b1) { mma16816(o[t][c], p[t], b0, b1); });
    }
    if constexpr (kFar) {
      if (far) {
#pragma unroll 1
        for (float top = kNear, up = 38.f; top > -130.f; top -= 20.f, up += 20.f) {
          const float down = ex2(-up);
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t p[MT][4];
            weigh(x, vf, n, seen, [&](int, int, float y, float) { return y >= top - 20.f && y < top ? ex2(y + up) : 0.f; }, p);
            if (__any_sync(0xffffffffu, (p[0][0] | p[0][2]) != 0))
              products(v_base, key + 8 * n, [&](int c, int t, uint32_t b0, uint32_t b1) {
                float x[4] = {};
                mma16816(x, p[t], b0, b1);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][c][i] = fmaf(x[i], down, o[t][c][i]);
              });
          }
        }
      }
    }
  }

  // A V scale of vtop or more: the next power of two above the largest, and the sums so far brought to it.
  static __device__ __noinline__ float next_vtop(float vtop, float most) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const uint32_t e = min((__float_as_uint(most) & 0x7f800000u) + (1u << 23), 252u << 23);
    return fmaxf(vtop, __uint_as_float(e));
  }
  __device__ __forceinline__ void raise_v(float most) {
    const float to = next_vtop(vtop, most), c = vtop / to;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][n][i] *= c;
    vtop = to;
  }

  // Weights of 16 keys as an operand; take(t, r, exponent, 2^exponent) gives a seen position's weight before V's scale.
  template <int NT, typename S, typename W>
  __device__ __forceinline__ void weigh(const float (&x)[MT][kPer][NT][2], const float (&vf)[NT][2], int n, S&& seen,
                                        W&& take, uint32_t (&p)[MT][4]) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
          float w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float y = x[t][r][n + h][i];
            w[i] = 0.f;
            if (seen(t, r, n + h, i)) {
              w[i] = take(t, r, y, ex2(y));
              if constexpr (F != kKvF16) w[i] *= vf[n + h][i];
            }
          }
          const __half2 lead = __floats2half2_rn(w[0], w[1]);
          p[t][2 * h + r] = half2_bits(lead);
          if constexpr (FOLD) {
            const float2 z = __half22float2(lead);
            p[t][2 * h + 1] = half2_bits(__floats2half2_rn(w[0] - z.x, w[1] - z.y));
          }
        }
  }

  // The V operands of 16 keys: use(c, t, b0, b1) for every output tile c and row tile t.
  template <typename U>
  __device__ __forceinline__ void products(uint32_t v_base, int key, U&& use) {
    const int lane = threadIdx.x & 31, mi = lane >> 3, r8 = lane & 7;
#pragma unroll
    for (int c = 0; c < kPieces; c += 2) {
      uint32_t w[4];
      ldsm4t(w, piece<F, HD, KEYS>(v_base, key + 8 * (mi & 1) + r8, c + (mi >> 1)));
      if constexpr (F == kKvF16) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          use(c, t, w[0], w[1]);
          use(c + 1, t, w[2], w[3]);
        }
      } else {  // a piece holds 16 dimensions: its even ones are tile 2 c, its odd ones tile 2 c + 1
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t e0, e1, d0, d1;
          unpack<F, true>(w[2 * j], e0, d0);
          unpack<F, true>(w[2 * j + 1], e1, d1);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            use(2 * (c + j), t, e0, e1);
            use(2 * (c + j) + 1, t, d0, d1);
          }
        }
      }
    }
  }

  // The row sums with V's power of two put back; l summed over the lanes of a row.
  __device__ __forceinline__ void finish() {
    const float up = F == kKvF16 ? 1.f : 0.5f * vtop;
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
  int64_t slot;      // item + CTA
  int own;
  int z, kvh, rt;    // plane of the cache; kv head, row tile
  int seq;           // own items: the sequence
  int t0, t1;        // units of this CTA
  int limit;         // positions that some row of the item sees
  int fewest;        // positions that every row sees
};

// The first unit of CTA c: the first total % grid CTAs take one unit more than the others.
__device__ __forceinline__ int share_start(int c, int total, int grid) {
  const int each = total / grid;
  return c * each + min(c, total - each * grid);
}
// The CTA that holds unit u < total.
__device__ __forceinline__ int share_of(int u, int total, int grid) {
  const int each = total / grid, more = total - each * grid, split = more * (each + 1);
  return u < split ? u / (each + 1) : more + (u - split) / each;
}

struct Walk {
  int u, end, b;
  Walk() = default;
  __device__ Walk(const Plan& p, const PrefixAttnArgs& a, const int32_t* cum) : b(0) {
    const int prefix = p.prefix_items * p.prefix_units, per = (int)a.own.heads * p.own_nrt;
    const int total = prefix + (per ? cum[a.B] * per : 0);
    u = share_start(blockIdx.x, total, gridDim.x);
    end = share_start(blockIdx.x + 1, total, gridDim.x);
    if (end > prefix) {  // the last sequence whose units start at or before the first own unit
      const int first = max(u - prefix, 0);
      int lo = 0, hi = (int)a.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (cum[mid] * per <= first) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
    }
  }
  __device__ __forceinline__ bool next(Piece& x, const Plan& p, const PrefixAttnArgs& a, const int32_t* cum) {
    if (u >= end) return false;
    const int prefix = p.prefix_items * p.prefix_units;
    int in, units;
    if (u >= prefix) {
      const int per = (int)a.own.heads * p.own_nrt, v = u - prefix;
      while (cum[b + 1] * per <= v) ++b;
      units = cum[b + 1] - cum[b];
      const int rest = v - cum[b] * per, j = rest / units;
      in = rest - j * units;
      x.slot = p.prefix_items + (int64_t)b * per + j;
      x.own = 1;
      x.kvh = j / p.own_nrt;
      x.rt = j % p.own_nrt;
      x.seq = b;
      x.z = b * (int)a.own.heads + x.kvh;
      const int first = x.rt * p.rt / p.G, last = (min((x.rt + 1) * p.rt, p.own_rows) - 1) / p.G;  // tokens
      const int seen = own_length(a, b, false) - (int)a.T + 1;
      x.limit = seen + last;
      x.fewest = seen + first;
    } else {
      units = p.prefix_units;
      x.slot = u / units;
      in = u - (int)x.slot * units;
      x.own = 0;
      x.kvh = (int)x.slot / p.prefix_nrt;
      x.rt = (int)x.slot % p.prefix_nrt;
      x.seq = 0;
      x.z = x.kvh;
      x.limit = x.fewest = (int)a.prefix_len;
    }
    const int n = min(units - in, end - u);
    x.t0 = in;
    x.t1 = in + n;
    x.slot += blockIdx.x;
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

// After a copy that was late: time for what is in flight to land before the shared memory is reused.
__device__ __noinline__ void grace() {
  const long long t0 = clock64();
  while (clock64() - t0 < 20000000LL) {}
}

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

// The sequences' unit counts, summed: cum[b] units of one row tile and kv head lie before sequence b.  Every CTA sums
// up to kMaxScan sequences itself; CTA 0 leaves the sums for the joining kernel.
__device__ const int32_t* unit_sums(const PrefixAttnArgs& a, const Plan& p, const int32_t* given, int32_t* shared,
                                    int32_t* out) {
  if (given || p.own_nrt == 0) return given;
  const int t = threadIdx.x, lane = t & 31;
  if (t < 32) {
    int sum = 0;
    for (int b0 = 0; b0 < (int)a.B; b0 += 32) {
      const int b = b0 + lane;
      int n = b < a.B ? (own_length(a, b, blockIdx.x == 0) + p.unit - 1) / p.unit : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += y;
      }
      if (b < a.B) {
        shared[b + 1] = sum + n;
        if (blockIdx.x == 0) out[b + 1] = sum + n;
      }
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) {
      shared[0] = 0;
      if (blockIdx.x == 0) out[0] = 0;
    }
  }
  return shared;
}

// q row of logical row `row` of an item (null past the end) and the positions it sees.
template <typename Q>
__device__ __forceinline__ const Q* q_row(const PrefixAttnArgs& a, const Plan& p, const Piece& x, int row, int& lim) {
  const int rho = x.rt * p.rt + row;
  if (rho >= (x.own ? p.own_rows : p.prefix_rows)) {
    lim = 0;
    return nullptr;
  }
  const int64_t b = x.own ? x.seq : rho / p.own_rows;
  const int in = x.own ? rho : rho % p.own_rows;
  const int t = in / p.G, g = in % p.G;
  lim = x.own ? x.fewest + t - x.rt * p.rt / p.G : x.limit;
  return static_cast<const Q*>(a.q) + b * a.qs.batch + t * a.qs.token + ((int64_t)x.kvh * p.G + g) * a.qs.head;
}

// A power of two that brings the largest of a folded row into [1, 2): its exponent leaves through the score factor, so
// that neither part of the split overflows or loses bits.  bits: max |q|; returns 2^-e.
__device__ __forceinline__ float row_shrink(uint32_t bits) {
  const uint32_t e = min(max(bits & 0x7f800000u, 64u << 23), 190u << 23);
  return __uint_as_float(0x7f000000u - e);
}

// Rows of the last tile past the end of the cached positions hold other data: V of f16 and e4m3 may be NaN there.
template <int F, int HD, int KEYS>
__device__ __forceinline__ void zero_v(uint8_t* v, int from, int to, int thread, int threads) {
  using Gm = Tile<F, HD, KEYS>;
  constexpr int kPer = Gm::kPart / 16;
  for (int i = thread; i < (to - from) * kPer * Gm::kBoxes; i += threads) {
    const int box = i / ((to - from) * kPer), j = i % ((to - from) * kPer);
    *reinterpret_cast<uint4*>(v + box * Gm::kBoxBytes + (from + j / kPer) * Gm::kPart + (j % kPer) * 16) = make_uint4(0, 0, 0, 0);
  }
  umma::fence_proxy_async_smem();
}

// ---------------------------------------------------------------- narrow

// What a warp copies next: position `key` of piece x, up to `end`.  Kept in shared memory: it is used once a tile.
struct Ahead {
  Walk w;
  Piece x;
  int key, end;
};

template <int F, int HD>
struct NarrowShared {
  uint64_t full[kWarps][Narrow<F, HD>::kStages];
  Ahead ahead[kWarps];
  int abort;
  int where[kWarps];
  float ml[kWarps][16][2];
  int32_t cum[kMaxScan + 1];
};

template <int F, int HD, bool FOLD, typename Q>
__global__ void __launch_bounds__(32 * kWarps, kNarrowCtas)
    narrow_attn_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan p, const __grid_constant__ Maps maps,
                       const int32_t* given, int32_t* cum_out) {
  using N = Narrow<F, HD>;
  using Tl = typename N::Tl;
  constexpr int KEYS = N::kKeys, RT = FOLD ? 8 : 16, kPer = FOLD ? 1 : 2;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ NarrowShared<F, HD> sh;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, tq = lane & 3;
  if (t == 0) {
    for (int i = 0; i < kWarps; ++i)
      for (int j = 0; j < N::kStages; ++j) umma::mbar_init(&sh.full[i][j], F == kKvF16 ? 1 : 33);
    sh.abort = 0;
    umma::fence_barrier_init();
  }
  const int32_t* cum = unit_sums(a, p, given, sh.cum, cum_out);
  __syncthreads();
  uint8_t* tiles = smem + warp * N::kStages * N::kStage;
  float* scales = reinterpret_cast<float*>(smem + kWarps * N::kStages * N::kStage + warp * N::kScales);
  Ahead& ahead = sh.ahead[warp];
  if (lane == 0) {
    ahead.w = Walk(p, a, cum);
    ahead.key = ahead.end = 0;
  }
  __syncwarp();
  int issued = 0, done = 0;     // tiles copied and used by this warp: stage = count mod kStages
  // Copy the warp's next tile.  The stage is the one whose tile was used last, so at least one stage is free whenever
  // no tile is being worked on: the join at the end of a piece uses it.
  auto copy = [&]() {
    if (ahead.key >= ahead.end) {
      __syncwarp();
      if (lane == 0)  // tiles warp, warp + 4, ... of every piece
        while (ahead.key >= ahead.end && ahead.w.next(ahead.x, p, a, cum)) {
          ahead.key = ahead.x.t0 * N::kUnit + warp * KEYS;
          ahead.end = min(ahead.x.t1 * N::kUnit, ahead.x.limit);
        }
      __syncwarp();
      if (ahead.key >= ahead.end) return;
    }
    const int s = issued % N::kStages, z = ahead.x.z, pos = ahead.key;
    const bool own = ahead.x.own != 0;
    const KvCache& c = own ? a.own : a.prefix;
    __syncwarp();
    uint64_t* bar = &sh.full[warp][s];
    const uint32_t dst = umma::smem_u32(tiles + s * N::kStage);
    if (lane == 0) {
      umma::mbar_arrive_expect_tx(bar, 2 * Tl::kBytes);
      ahead.key = pos + kWarps * KEYS;
      const CUtensorMap *mk = own ? &maps.ok : &maps.pk, *mv = own ? &maps.ov : &maps.pv;
#pragma unroll
      for (int b = 0; b < Tl::kBoxes; ++b) {
        tma_load_3d(dst + b * Tl::kBoxBytes, mk, bar, b * (Tl::kPart / Tl::kEsz), pos, z);
        tma_load_3d(dst + Tl::kBytes + b * Tl::kBoxBytes, mv, bar, b * (Tl::kPart / Tl::kEsz), pos, z);
      }
    }
    if constexpr (F != kKvF16) {  // row scales: 4-byte copies, zero past the end of the cache
      const bool in = pos + lane < c.max_seq;
      const int64_t at = (int64_t)z * c.max_seq + (in ? pos + lane : 0);
      const uint32_t to = umma::smem_u32(scales + s * (2 * KEYS)) + 4 * lane;
      const int bytes = in ? 4 : 0;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(c.k_scale + at), "r"(bytes) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4 * KEYS), "l"(c.v_scale + at), "r"(bytes) : "memory");
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(umma::smem_u32(bar)) : "memory");
    }
    ++issued;
    __syncwarp();
  };
  for (int i = 0; i < N::kStages - 1; ++i) copy();

  Rows<F, HD, FOLD, 1, KEYS> st;
  const float base = a.scale * kLog2e;
  Walk w(p, a, cum);
  Piece x;
  while (w.next(x, p, a, cum)) {
    st.clear();
    uint32_t qa[HD / 16][4];
    const Q* src[2];
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      src[r] = q_row<Q>(a, p, x, g + 8 * r, st.lim[0][r]);
      st.f[0][r] = base;
    }
    float shrink = 1.f;
    if constexpr (FOLD && sizeof(Q) == 4) {
      uint32_t mx = 0;
      if (src[0])
#pragma unroll
        for (int d = 0; d < HD / 4; ++d) mx = max(mx, __float_as_uint((float)src[0][4 * d + tq]) & 0x7fffffffu);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      shrink = row_shrink(mx);
      st.f[0][0] = base / shrink;
    }
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // elements 2 tq, 2 tq + 1 (+ 8): dimensions 4 tq ... of K's words in bytes
        const int d = F == kKvF16 ? 16 * ks + 8 * h + 2 * tq : 16 * ks + 4 * tq + 2 * h;
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
          const float y0 = src[r] ? (float)src[r][d] * shrink : 0.f, y1 = src[r] ? (float)src[r][d + 1] * shrink : 0.f;
          const __half2 lead = __floats2half2_rn(y0, y1);
          qa[ks][2 * h + r] = half2_bits(lead);
          if constexpr (FOLD) {
            const float2 z = __half22float2(lead);
            qa[ks][2 * h + 1] = half2_bits(__floats2half2_rn(y0 - z.x, y1 - z.y));
          }
        }
      }
    const int end = min(x.t1 * N::kUnit, x.limit);
#pragma unroll 1
    for (int key = x.t0 * N::kUnit + warp * KEYS; key < end; key += kWarps * KEYS) {
      copy();
      const int s = done % N::kStages;
      umma::bounded_wait(&sh.full[warp][s], (done / N::kStages) & 1, &sh.abort, a.err, kErrKvCopy);
      uint8_t* stage = tiles + s * N::kStage;
      const uint32_t k_base = umma::smem_u32(stage);
      const int left = x.limit - key;
      if (F != kKvI8 && left < KEYS) {
        zero_v<F, HD, KEYS>(stage + Tl::kBytes, left, KEYS, lane, 32);
        __syncwarp();
      }
      const float* ks = scales + s * (2 * KEYS);
      auto frag = [&](int step, int, uint32_t (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = qa[step][i];
      };
      if (key + KEYS > x.fewest) st.template step<KEYS / 8, true>(k_base, k_base + Tl::kBytes, ks, ks + KEYS, 0, left, key, frag);
      else st.template step<KEYS / 8, false>(k_base, k_base + Tl::kBytes, ks, ks + KEYS, 0, left, key, frag);
      __syncwarp();
      ++done;
    }
    st.finish();
    // join the four warps' keys: each leaves its rows in its free stage
    const int free_stage = (done + N::kStages - 1) % N::kStages;
    float* mine = reinterpret_cast<float*>(tiles + free_stage * N::kStage);
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      st.store(mine + (g + 8 * r) * HD, 0, r);
      if (tq == 0) {
        sh.ml[warp][g + 8 * r][0] = st.m[0][r];
        sh.ml[warp][g + 8 * r][1] = st.l[0][r];
      }
    }
    if (lane == 0) sh.where[warp] = (int)(reinterpret_cast<uint8_t*>(mine) - smem);
    __syncthreads();
    float* part = p.part + x.slot * (RT * HD);
    float* ml = p.ml + x.slot * (RT * 2);
    for (int i = t; i < RT * HD / 4; i += 32 * kWarps) {
      const int row = i / (HD / 4);
      float mx = sh.ml[0][row][0];
#pragma unroll
      for (int k = 1; k < kWarps; ++k) mx = fmaxf(mx, sh.ml[k][row][0]);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = mx == -INFINITY ? 1.f : ex2(sh.ml[k][row][0] - mx);
        const float4 y = reinterpret_cast<const float4*>(smem + sh.where[k])[i];
        sum.x = fmaf(f, y.x, sum.x);
        sum.y = fmaf(f, y.y, sum.y);
        sum.z = fmaf(f, y.z, sum.z);
        sum.w = fmaf(f, y.w, sum.w);
        l = fmaf(f, sh.ml[k][row][1], l);
      }
      reinterpret_cast<float4*>(part)[i] = sum;
      if (i % (HD / 4) == 0) *reinterpret_cast<float2*>(ml + 2 * row) = make_float2(mx, l);
    }
    umma::fence_proxy_async_smem();  // the stages take copies again
    __syncthreads();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (*(volatile int*)&sh.abort) grace();
}

// ---------------------------------------------------------------- wide

template <int STAGES>
struct WideShared {
  uint64_t full[STAGES], empty[STAGES];
  int abort;
  float shrink[kWarps][16];
  int32_t cum[kMaxScan + 1];
};

template <int F, int HD, bool FOLD, typename Q, typename C>
__device__ void consume(const PrefixAttnArgs& a, const Plan& p, const int32_t* cum, uint8_t* smem, C& ctl) {
  using Wd = Wide<F, HD>;
  using Tl = typename Wd::Tl;
  constexpr int MT = 2;
  constexpr int RPT = FOLD ? 8 : 16;                       // logical rows of an MMA tile
  constexpr int RT = kWarps * MT * RPT;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, tq = lane & 3;
  uint8_t* share = smem + Wd::kStages * Wd::kStage;
  Ring ring(Wd::kStages);
  Rows<F, HD, FOLD, MT, kTile> st;
  const float base = a.scale * kLog2e;
  Walk w(p, a, cum);
  Piece x;
  while (w.next(x, p, a, cum)) {
    st.clear();
    // 128 operand rows of q in shared memory, 16-byte pieces swizzled, one thread a row
    const int tile = t >> 4, r = t & 15;                    // operand row t: MMA tile t / 16
    int lim;
    const Q* src = q_row<Q>(a, p, x, tile * RPT + (FOLD ? r & 7 : r), lim);
    float shrink = 1.f;
    if constexpr (FOLD) {
      uint32_t mx = 0;
      if (src)
        for (int d = 0; d < HD; ++d) mx = max(mx, __float_as_uint((float)src[d]) & 0x7fffffffu);
      shrink = row_shrink(mx);
      if (!(r & 8)) ctl.shrink[warp][(tile & 1) * 8 + (r & 7)] = shrink;
    }
    for (int c = 0; c < HD / 8; ++c) {  // the eight operand positions of piece c
      __half h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int d = 8 * c + i;                                  // operand position -> dimension
        if constexpr (F != kKvF16) d = (d & ~15) | ((d & 6) << 1) | ((d & 8) >> 2) | (d & 1);
        const float y = src ? (float)src[d] * shrink : 0.f;
        const __half lead = __float2half_rn(y);
        h[i] = FOLD && (r & 8) ? __float2half_rn(y - __half2float(lead)) : lead;
      }
      *reinterpret_cast<uint4*>(share + t * (2 * HD) + ((c ^ (t & 7)) << 4)) = *reinterpret_cast<const uint4*>(h);
    }
    compute_barrier();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r2 = 0; r2 < (FOLD ? 1 : 2); ++r2) {
        (void)q_row<Q>(a, p, x, (warp * MT + m) * RPT + g + 8 * r2, st.lim[m][r2]);
        st.f[m][r2] = FOLD ? base / ctl.shrink[warp][m * 8 + g] : base;
      }
    const int last = min(x.t1, (x.limit + kTile - 1) / kTile);
    for (int kt = x.t0; kt < last; ++kt) {
      umma::bounded_wait(&ctl.full[ring.stage], ring.phase, &ctl.abort, a.err, kErrKvCopy);
      uint8_t* stage = smem + ring.stage * Wd::kStage;
      const uint32_t k_base = umma::smem_u32(stage), v_base = k_base + Tl::kBytes;
      const float* ks = reinterpret_cast<const float*>(stage + 2 * Tl::kBytes);
      const int pos0 = kt * kTile, left = x.limit - pos0;
      const bool masked = pos0 + kTile > x.fewest;
      if (F != kKvI8 && left < kTile) {
        zero_v<F, HD, kTile>(stage + Tl::kBytes, left, kTile, t, 32 * kWarps);
        compute_barrier();
      }
      auto frag = [&](int step, int m, uint32_t (&f)[4]) {
        // matrices: rows 0-7 and 8-15 of the tile, pieces 2 step and 2 step + 1
        const int row = (warp * MT + m) * 16 + (lane & 15), c = 2 * step + (lane >> 4);
        ldsm4(f, umma::smem_u32(share) + row * (2 * HD) + ((c ^ (row & 7)) << 4));
      };
#pragma unroll 1
      for (int key = 0; key < kTile; key += 32) {
        if (masked) st.template step<4, true>(k_base, v_base, ks, ks + kTile, key, left, pos0, frag);
        else st.template step<4, false>(k_base, v_base, ks, ks + kTile, key, left, pos0, frag);
      }
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(&ctl.empty[ring.stage]);
      ring.advance();
    }
    compute_barrier();  // q's rows and scales are free again
    st.finish();
    float* part = p.part + x.slot * (RT * HD);
    float* ml = p.ml + x.slot * (RT * 2);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r2 = 0; r2 < (FOLD ? 1 : 2); ++r2) {
        const int row = (warp * MT + m) * RPT + g + 8 * r2;
        st.store(part + (int64_t)row * HD, m, r2);
        if (tq == 0) *reinterpret_cast<float2*>(ml + 2 * row) = make_float2(st.m[m][r2], st.l[m][r2]);
      }
  }
}

template <int F, int HD, typename C>
__device__ void produce(const PrefixAttnArgs& a, const Plan& p, const Maps& maps, const int32_t* cum, uint8_t* smem, C& ctl) {
  using Wd = Wide<F, HD>;
  using Tl = typename Wd::Tl;
  const int lane = threadIdx.x & 31;
  Ring ring(Wd::kStages);
  Walk w(p, a, cum);
  Piece x;
  while (w.next(x, p, a, cum)) {
    const KvCache& c = x.own ? a.own : a.prefix;
    const CUtensorMap *mk = x.own ? &maps.ok : &maps.pk, *mv = x.own ? &maps.ov : &maps.pv;
    const int last = min(x.t1, (x.limit + kTile - 1) / kTile);
    for (int kt = x.t0; kt < last; ++kt) {
      const bool ok = umma::bounded_wait(&ctl.empty[ring.stage], ring.phase ^ 1, &ctl.abort, a.err, kErrKvCopy);
      if (!ok) return;
      uint8_t* stage = smem + ring.stage * Wd::kStage;
      uint64_t* bar = &ctl.full[ring.stage];
      if (lane == 0) {
        umma::mbar_arrive_expect_tx(bar, 2 * Tl::kBytes);
        const uint32_t dst = umma::smem_u32(stage);
#pragma unroll
        for (int b = 0; b < Tl::kBoxes; ++b) {
          tma_load_3d(dst + b * Tl::kBoxBytes, mk, bar, b * (Tl::kPart / Tl::kEsz), kt * kTile, x.z);
          tma_load_3d(dst + Tl::kBytes + b * Tl::kBoxBytes, mv, bar, b * (Tl::kPart / Tl::kEsz), kt * kTile, x.z);
        }
      }
      if constexpr (F != kKvF16) {  // row scales: 4-byte copies, zero past the end of the cache
        const uint32_t dst = umma::smem_u32(stage + 2 * Tl::kBytes);
#pragma unroll
        for (int i = 0; i < 2 * kTile / 32; ++i) {
          const int j = (i % (kTile / 32)) * 32 + lane;
          const int64_t pos = (int64_t)kt * kTile + j;
          const bool in = pos < c.max_seq;
          const float* src = (i < kTile / 32 ? c.k_scale : c.v_scale) + (int64_t)x.z * c.max_seq + (in ? pos : 0);
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

template <int F, int HD, typename Q>
__global__ void __launch_bounds__(32 * (kWarps + 1), kWideCtas)
    wide_attn_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan p, const __grid_constant__ Maps maps,
                     const int32_t* given, int32_t* cum_out) {
  using Wd = Wide<F, HD>;
  constexpr bool kFold = sizeof(Q) == 4;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ WideShared<Wd::kStages> ctl;
  const int t = threadIdx.x;
  if (t == 0) {
    for (int i = 0; i < Wd::kStages; ++i) {
      umma::mbar_init(&ctl.full[i], F == kKvF16 ? 1 : 33);
      umma::mbar_init(&ctl.empty[i], kWarps);
    }
    ctl.abort = 0;
    umma::fence_barrier_init();
  }
  const int32_t* cum = unit_sums(a, p, given, ctl.cum, cum_out);
  __syncthreads();
  if (t >= 32 * kWarps) produce<F, HD>(a, p, maps, cum, smem, ctl);
  else consume<F, HD, kFold, Q>(a, p, cum, smem, ctl);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (*(volatile int*)&ctl.abort) grace();
}

// Units of the sequences before each, for batches too large for a CTA's shared memory.
__global__ void __launch_bounds__(1024) unit_sums_kernel(const __grid_constant__ PrefixAttnArgs a, int unit, int32_t* cum) {
  __shared__ int warp_sum[32];
  const int t = threadIdx.x, lane = t & 31;
  int before = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += 1024) {
    const int64_t b = b0 + t;
    int n = b < a.B ? (own_length(a, b, true) + unit - 1) / unit : 0;
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

// out = sum over a row's pieces of 2^(m - M) o / sum of 2^(m - M) l, prefix pieces first.  One warp per row.  px, po:
// the plans of the kernels that took the prefix and the own items.
template <int HD, typename Q>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan px,
                                                   const __grid_constant__ Plan po, const int32_t* __restrict__ cum) {
  constexpr int N = HD / 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= a.B * a.T * a.H) return;
  const int64_t h = row % a.H, bt = row / a.H, b = bt / a.T, t = bt % a.T;
  const int64_t kvh = h / po.G, g = h % po.G;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the pieces are there from here on
  float mx = -INFINITY, l = 0.f, o[N] = {};
#pragma unroll 1
  for (int own = px.prefix_items ? 0 : 1; own < 2; ++own) {
    const Plan& p = own ? po : px;
    const int rho = (int)(own ? t * p.G + g : bt * p.G + g), j = rho / p.rt, in = rho - j * p.rt;
    const int per = (int)a.own.heads * p.own_nrt, prefix = p.prefix_items * p.prefix_units;
    const int total = prefix + (per ? cum[a.B] * per : 0);
    int64_t item;
    int u0, units;
    if (own) {
      units = cum[b + 1] - cum[b];
      item = p.prefix_items + b * per + kvh * p.own_nrt + j;
      u0 = prefix + cum[b] * per + ((int)kvh * p.own_nrt + j) * units;
    } else {
      units = p.prefix_units;
      item = kvh * p.prefix_nrt + j;
      u0 = (int)item * units;
    }
    if (units == 0) continue;
    const int first = share_of(u0, total, p.grid), last = share_of(u0 + units - 1, total, p.grid);
    for (int c = first; c <= last; ++c) {
      const int64_t r = (item + c) * p.rt + in;
      const float2 ml = *reinterpret_cast<const float2*>(p.ml + 2 * r);
      const float* src = p.part + r * HD + N * lane;
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

// [batch * heads, max_seq, hd] as boxes of `keys` positions of at most 128 bytes; positions past max_seq read as zero.
bool make_map(CUtensorMap* map, const KvCache& c, const void* data, int keys) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t esz = c.fmt == kKvF16 ? 2 : 1, row = esz * c.hd;
  const cuuint32_t span = (cuuint32_t)(row < 128 ? row : 128);
  const cuuint64_t dims[3] = {(cuuint64_t)c.hd, (cuuint64_t)c.max_seq, (cuuint64_t)(c.batch * c.heads)};
  const cuuint64_t strides[2] = {row, row * (cuuint64_t)c.max_seq};
  const cuuint32_t box[3] = {(cuuint32_t)(span / esz), (cuuint32_t)keys, 1}, es[3] = {1, 1, 1};
  return enc(map, c.fmt == kKvF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
             const_cast<void*>(data), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

int narrow_keys(const PrefixAttnArgs& a) { return a.own.fmt == kKvF16 && a.own.hd == 128 ? 16 : 32; }

// Which kernel takes the prefix and which the own items, their plans, and the workspace.
struct Layout {
  Plan narrow, wide;
  bool prefix_wide = false, own_wide = false;
  size_t bytes = 0;
  int64_t most = 0;  // units of either kernel, at most
  const Plan& of_prefix() const { return prefix_wide ? wide : narrow; }
  const Plan& of_own() const { return own_wide ? wide : narrow; }
};

Layout lay_out(const PrefixAttnArgs& a, char* ws) {
  Layout l{};
  const int G = (int)(a.H / a.own.heads);
  const int own_rows = (int)(a.T * G), prefix_rows = (int)(a.B * own_rows);
  l.own_wide = own_rows > 16;
  l.prefix_wide = a.prefix_len && prefix_rows > 16;
  size_t used = up256(sizeof(int32_t) * (size_t)(a.B + 1));
  for (int w = 0; w < 2; ++w) {
    Plan& p = w ? l.wide : l.narrow;
    const bool prefix = a.prefix_len && l.prefix_wide == (w != 0), own = l.own_wide == (w != 0);
    p.G = G;
    p.own_rows = own_rows;
    p.prefix_rows = prefix_rows;
    p.rt = w ? (a.half ? 128 : 64) : a.half && (prefix ? prefix_rows : own_rows) > 8 ? 16 : 8;
    p.unit = w ? kTile : kWarps * narrow_keys(a);
    p.own_nrt = own ? (own_rows + p.rt - 1) / p.rt : 0;
    p.prefix_nrt = prefix ? (prefix_rows + p.rt - 1) / p.rt : 0;
    p.prefix_units = prefix ? (int)((a.prefix_len + p.unit - 1) / p.unit) : 0;
    p.prefix_items = (int)a.own.heads * p.prefix_nrt;
    const int64_t own_items = a.B * a.own.heads * p.own_nrt;
    const int64_t most = (int64_t)p.prefix_items * p.prefix_units + own_items * ((a.own.max_seq + p.unit - 1) / p.unit);
    l.most = most > l.most ? most : l.most;
    const int full = kSms * (w ? kWideCtas : kNarrowCtas);
    p.grid = (int)(most < full ? most : full);
    if (p.grid == 0) continue;
    const int64_t rows = (p.prefix_items + own_items + p.grid) * p.rt;
    p.part = reinterpret_cast<float*>(ws + used);
    used += up256(sizeof(float) * (size_t)(rows * a.own.hd));
    p.ml = reinterpret_cast<float*>(ws + used);
    used += up256(sizeof(float) * (size_t)(rows * 2));
  }
  l.bytes = used;
  return l;
}

template <typename K>
cudaError_t run(K kern, int smem, int threads, const PrefixAttnArgs& a, const Plan& p, const Maps& maps, const int32_t* given,
                int32_t* cum, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)p.grid, threads, smem, st>>>(a, p, maps, given, cum);
  return cudaGetLastError();
}

bool make_maps(Maps* m, const PrefixAttnArgs& a, int keys) {
  return make_map(&m->ok, a.own, a.own.k, keys) && make_map(&m->ov, a.own, a.own.v, keys) &&
         (!a.prefix_len || (make_map(&m->pk, a.prefix, a.prefix.k, keys) && make_map(&m->pv, a.prefix, a.prefix.v, keys)));
}

template <int F, int HD>
cudaError_t run_all(const PrefixAttnArgs& a, const Layout& l, const int32_t* given, int32_t* cum, cudaStream_t st) {
  Maps maps;
  if (l.wide.grid) {
    if (!make_maps(&maps, a, kTile)) return cudaErrorInvalidValue;
    constexpr int smem = Wide<F, HD>::kSmem, threads = 32 * (kWarps + 1);
    const cudaError_t e = a.half ? run(wide_attn_kernel<F, HD, __half>, smem, threads, a, l.wide, maps, given, cum, st)
                                 : run(wide_attn_kernel<F, HD, float>, smem, threads, a, l.wide, maps, given, cum, st);
    if (e != cudaSuccess) return e;
  }
  if (l.narrow.grid) {
    if (!make_maps(&maps, a, Narrow<F, HD>::kKeys)) return cudaErrorInvalidValue;
    constexpr int smem = Narrow<F, HD>::kSmem, threads = 32 * kWarps;
    const Plan& p = l.narrow;
    const cudaError_t e = !a.half       ? run(narrow_attn_kernel<F, HD, true, float>, smem, threads, a, p, maps, given, cum, st)
                          : p.rt == 16 ? run(narrow_attn_kernel<F, HD, false, __half>, smem, threads, a, p, maps, given, cum, st)
                                       : run(narrow_attn_kernel<F, HD, true, __half>, smem, threads, a, p, maps, given, cum, st);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((a.B * a.T * a.H + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const int32_t* sums = cum;
  return a.half ? cudaLaunchKernelEx(&cfg, join_kernel<HD, __half>, a, l.of_prefix(), l.of_own(), sums)
                : cudaLaunchKernelEx(&cfg, join_kernel<HD, float>, a, l.of_prefix(), l.of_own(), sums);
}

template <int F>
cudaError_t run_dim(const PrefixAttnArgs& a, const Layout& l, const int32_t* given, int32_t* cum, cudaStream_t st) {
  return a.own.hd == 128 ? run_all<F, 128>(a, l, given, cum, st) : run_all<F, 64>(a, l, given, cum, st);
}

}  // namespace

size_t prefix_attn_ws(const PrefixAttnArgs& a) { return lay_out(a, nullptr).bytes; }

cudaError_t launch_prefix_attn(const PrefixAttnArgs& a, void* ws, int* launches, cudaStream_t st) {
  const Layout l = lay_out(a, static_cast<char*>(ws));
  if (l.most >= (int64_t(1) << 30)) return cudaErrorInvalidValue;  // (a cache of 2^36 positions)
  int32_t* cum = static_cast<int32_t*>(ws);
  const int32_t* given = nullptr;
  *launches = 1 + (l.wide.grid > 0) + (l.narrow.grid > 0);
  if (a.B > kMaxScan) {
    unit_sums_kernel<<<1, 1024, 0, st>>>(a, l.of_own().unit, cum);
    given = cum;
    ++*launches;
  }
  if (a.own.fmt == kKvI8) return run_dim<kKvI8>(a, l, given, cum, st);
  if (a.own.fmt == kKvE4M3) return run_dim<kKvE4M3>(a, l, given, cum, st);
  return run_dim<kKvF16>(a, l, given, cum, st);
}

}  // namespace uaii_b200
