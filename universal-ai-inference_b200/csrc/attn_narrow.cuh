// attn_narrow.cuh -- attention items of at most 8 or 16 rows on warp-level MMAs (see prefix_attn.cu).
#pragma once

#include "attn_common.cuh"

namespace uaii_b200 {
namespace attn {

// Narrow: every warp is a worker of its own, with its own copies: kKeys positions at a time, the next ones while it
// works.  Three CTAs of four warps hold 200 KB of an SM, about half of it in flight.
// A step of 32 keys of 128 dimensions takes a warp about 780 instructions (bytes to f16 a third of them); 32 sequences
// around 4096 i8 positions (275 MB) take 51.5 us, 5.3 TB/s, 0.83 of a copy's rate, at half the issue rate: a warp's chain
// from copied bytes over scores and weights to sums is what it waits for.  A further piece costs a warp about 7000 cycles.
template <int F, int HD>
struct Narrow {
  static constexpr int kKeys = F == kKvF16 && HD == 128 ? 16 : 32;
  using Tl = Tile<F, HD, kKeys>;
  static constexpr int kStage = 2 * Tl::kBytes;             // 4, 8 or (f16 of 16 keys) 8 KB
  static constexpr int kStages = 16 * 1024 / kStage;
  static constexpr int kScales = kStages * Tl::kScaleBytes; // of one warp, after all the tiles
  static constexpr int kSmem = kWarps * (kStages * kStage + kScales) + 1024;
};

// ---------------------------------------------------------------- one warp's running softmax

template <int F, int HD, bool FOLD, int KEYS, bool F32>
struct Rows {
  static constexpr int kPer = FOLD ? 1 : 2;  // logical rows of a lane in one MMA tile
  static constexpr int kPieces = HD * Tile<F, HD, KEYS>::kEsz / 16;  // 16-byte pieces of a row
  // The two parts of a weight resolve 2^-24, f16's smallest step (2^-33 of the largest).  Smaller weights are added in passes
  // of their own, 20 binary orders at a time, raised to [2^-6, 2^14): only very uneven scores (22 e-foldings) need them.
  static constexpr bool kFar = FOLD;
  static constexpr float kNear = 0x1p-24f;
  float o[HD / 8][4];
  float m[kPer], l[kPer];  // the reference (attn_common.cuh), the denominator
  float f[kPer];           // score factor: scale * log2(e), and the power of two taken out of a folded row of q
  int lim[kPer];           // positions the row sees
  // The tensor cores cut sums off where they should round (half of f32's last place at each addition: 1e-5 of a sum was
  // measured after the 650 of 320 steps), so f32 sums are taken out after 32 additions and added up in f32.
  static constexpr bool kTake = FOLD && F32;
  static constexpr int kTakeSteps = 32 / (KEYS / 16);
  float taken_m;           // their reference

  // Leading part and rest.  Where an f16 cache holds an infinity, the rest is 0 * inf.
  static __device__ __forceinline__ float join(float lead, float rest) {
    if constexpr (F == kKvF16) return fabsf(lead) == INFINITY ? lead : lead + rest;
    return lead + rest;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    taken_m = -INFINITY;
  }

  // Keys [key, key + 8 NT) of the tile at k_base / v_base, which starts at position pos0; masked says that some row may not
  // see all of them.  a(ks, frag) gives the query operands.
  template <int NT, bool masked, typename A>
  __device__ __forceinline__ void step(uint32_t k_base, uint32_t v_base, const float* ks, const float* vs, int key, int pos0, A&& a) {
    const int lane = threadIdx.x & 31, tq = lane & 3, mi = lane >> 3, r8 = lane & 7;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
    // scores: four 16-byte pieces of eight keys at a time
#pragma unroll
    for (int c = 0; c < kPieces; c += 4) {
      constexpr int kSteps = F == kKvF16 ? 2 : 4;
      uint32_t q[kSteps][4];
#pragma unroll
      for (int j = 0; j < kSteps; ++j) a((F == kKvF16 ? c / 2 : c) + j, q[j]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t w[4];
        ldsm4(w, piece<F, HD, KEYS>(k_base, key + 8 * n + r8, c + mi));
        if constexpr (F == kKvF16) {
          mma16816(s[n], q[0], w[0], w[1]);
          mma16816(s[n], q[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t b0, b1;
            unpack<F, false>(w[j], b0, b1);
            mma16816(s[n], q[j], b0, b1);
          }
        }
      }
    }
    // columns 2 tq, 2 tq + 1 of each eight keys: K and V scales
    float kf[NT][2], vf[NT][2], large = 0.f;  // log2 of this lane's largest V scale
    if constexpr (F != kKvF16) {
      float most = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 x = *reinterpret_cast<const float2*>(ks + key + 8 * n + 2 * tq);
        const float2 y = *reinterpret_cast<const float2*>(vs + key + 8 * n + 2 * tq);
        kf[n][0] = x.x; kf[n][1] = x.y;
        vf[n][0] = y.x; vf[n][1] = y.y;
        most = fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y)));  // (a NaN shows in its products, not here)
      }
      large = log2_scale(most);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if constexpr (FOLD) s[n][i] = join(s[n][i], s[n][2 + i]);
    auto seen = [&](int r, int n, int i) { return !masked || pos0 + key + 8 * n + 2 * tq + i < lim[r]; };
    auto factor = [&](int r, int n, int i) {
      if constexpr (F == kKvF16) return f[r];
      else return kf[n][i] * f[r];
    };
    // exponents against the reference as it is; a lane checks its own, and a row's maxima are only made when a product may
    // be too large
    float x[kPer][NT][2];
    bool over = false;
    auto exponents = [&](int r) {
      const float off = kLift - (m[r] == -INFINITY ? 0.f : m[r]);
      float most = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[r][n][i] = fmaf(s[n][2 * r + i], factor(r, n, i), off);
          if (seen(r, n, i)) most = fmaxf(most, x[r][n][i]);
        }
      over |= most + large > kMostProduct || most > kMostWeight || (m[r] == -INFINITY && most > -INFINITY);
    };
#pragma unroll
    for (int r = 0; r < kPer; ++r) exponents(r);
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        float top = -INFINITY, product = -INFINITY;  // the largest score, the largest product
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (seen(r, n, i)) {
              const float y = s[n][2 * r + i] * factor(r, n, i);
              top = fmaxf(top, y);
              if constexpr (F != kKvF16) product = fmaxf(product, y + log2_scale(vf[n][i]));
            }
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          if constexpr (F != kKvF16) product = fmaxf(product, __shfl_xor_sync(0xffffffffu, product, d));
        }
        const float to = next_reference(m[r], top, F == kKvF16 ? top : product);
        const float c = to > m[r] ? ex2(m[r] - to) : 1.f;
        m[r] = to;
        l[r] *= c;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          o[n][2 * r] *= c;
          o[n][2 * r + 1] *= c;
          if constexpr (FOLD) {
            o[n][2] *= c;
            o[n][3] *= c;
          }
        }
        exponents(r);
      }
    }
    // a seen position's weight times its V scale
    auto weight = [&](int r, int n, int i, float& e) {
      e = ex2(x[r][n][i]);
      if constexpr (F == kKvF16) return e;
      else return e * vf[n][i];
    };
    float low = 1.f;  // the smallest
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t p[4], rest[4];
      operand(n, [&](int r, int n, int i) {
        if (!seen(r, n, i)) return 0.f;
        float e;
        const float w = weight(r, n, i, e);
        l[r] += e;
        if (kFar) low = fminf(low, w);
        return kFar && w < kNear ? 0.f : w;
      }, p, rest);
      products(v_base, key + 8 * n, [&](int c, uint32_t b0, uint32_t b1) {
        mma16816(o[c], p, b0, b1);
        if constexpr (!FOLD) mma16816(o[c], rest, b0, b1);
      });
    }
    if constexpr (kFar) {
      if (__any_sync(0xffffffffu, low < kNear)) {
#pragma unroll 1
        for (float top = kNear, up = 0x1p38f, down = 0x1p-38f; top > 0x1p-110f; top *= 0x1p-20f, up *= 0x1p20f, down *= 0x1p-20f) {
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t p[4], rest[4];
            operand(n, [&](int r, int n, int i) {
              float e;
              const float w = weight(r, n, i, e);
              return seen(r, n, i) && w >= top * 0x1p-20f && w < top ? w * up : 0.f;
            }, p, rest);
            if (__any_sync(0xffffffffu, (p[0] | p[2]) != 0))
              products(v_base, key + 8 * n, [&](int c, uint32_t b0, uint32_t b1) {
                float y[4] = {};
                mma16816(y, p, b0, b1);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][i] = fmaf(y[i], down, o[c][i]);
              });
          }
        }
      }
    }
  }

  // Weights of 16 keys, weight(r, n, i), as an operand: leading parts, and what their rounding left, in rows of its own (FOLD)
  // or as a second operand.
  template <typename W>
  __device__ __forceinline__ void operand(int n, W&& weight, uint32_t (&p)[4], uint32_t (&rest)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        const float x = weight(r, n + h, 0), y = weight(r, n + h, 1);
        split_weights<F == kKvF16 && !FOLD>(x, y, p[2 * h + r], FOLD ? p[2 * h + 1] : rest[2 * h + r]);
      }
  }

  // The V operands of 16 keys: use(c, b0, b1) for every output tile c.
  template <typename U>
  __device__ __forceinline__ void products(uint32_t v_base, int key, U&& use) {
    const int lane = threadIdx.x & 31, mi = lane >> 3, r8 = lane & 7;
#pragma unroll
    for (int c = 0; c < kPieces; c += 2) {
      uint32_t w[4];
      ldsm4t(w, piece<F, HD, KEYS>(v_base, key + 8 * (mi & 1) + r8, c + (mi >> 1)));
      if constexpr (F == kKvF16) {
        use(c, w[0], w[1]);
        use(c + 1, w[2], w[3]);
      } else {  // a piece holds 16 dimensions: its even ones are tile 2 c, its odd ones tile 2 c + 1
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t e0, e1, d0, d1;
          unpack<F, true>(w[2 * j], e0, d0);
          unpack<F, true>(w[2 * j + 1], e1, d1);
          use(2 * (c + j), e0, e1);
          use(2 * (c + j) + 1, d0, d1);
        }
      }
    }
  }

  // Row r's sums to dst[HD], added to those taken out before (`more`); the next ones start from nothing.
  __device__ __forceinline__ void take_out(float* dst, int r, bool more) {
    const int tq = threadIdx.x & 3;
    const float old = taken_m == m[r] ? 1.f : ex2(taken_m - m[r]);
    auto out = [&](int n, int i) {
      float y = o[n][2 * r + i];
      if constexpr (FOLD) y = join(y, o[n][2 + i]);
      o[n][2 * r + i] = 0.f;
      if constexpr (FOLD) o[n][2 + i] = 0.f;
      return y;
    };
    if constexpr (F == kKvF16) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        float2* at = reinterpret_cast<float2*>(dst + 8 * n + 2 * tq);
        float2 y = make_float2(out(n, 0), out(n, 1));
        if (kTake && more) {
          const float2 z = *at;
          y = make_float2(fmaf(z.x, old, y.x), fmaf(z.y, old, y.y));
        }
        *at = y;
      }
    } else {
#pragma unroll
      for (int n = 0; n < HD / 8; n += 2) {
        float4* at = reinterpret_cast<float4*>(dst + 8 * n + 4 * tq);
        float4 y = make_float4(out(n, 0), out(n + 1, 0), out(n, 1), out(n + 1, 1));
        if (kTake && more) {
          const float4 z = *at;
          y = make_float4(fmaf(z.x, old, y.x), fmaf(z.y, old, y.y), fmaf(z.z, old, y.z), fmaf(z.w, old, y.w));
        }
        *at = y;
      }
    }
    taken_m = m[r];
  }

  // Row r's denominator, summed over its lanes.
  __device__ __forceinline__ float denominator(int r) const {
    float y = l[r];
    y += __shfl_xor_sync(0xffffffffu, y, 1);
    return y + __shfl_xor_sync(0xffffffffu, y, 2);
  }
};

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

// V of positions that only some of an item's tokens see: infinities and NaNs (which an 8-bit integer is not) become
// zeros, since 0 times either would reach the tokens that do not see them, and the joining kernel gives them to those
// that do.  Whether there was one, for the whole warp.
template <int F, int HD, int KEYS>
__device__ __noinline__ bool hide_v(uint8_t* v, int from, int to, int lane) {
  using Gm = Tile<F, HD, KEYS>;
  constexpr int kPer = Gm::kPart / 16;
  bool any = false;
  for (int i = lane; i < (to - from) * kPer * Gm::kBoxes; i += 32) {
    const int box = i / ((to - from) * kPer), j = i % ((to - from) * kPer);
    uint4* at = reinterpret_cast<uint4*>(v + box * Gm::kBoxBytes + (from + j / kPer) * Gm::kPart + (j % kPer) * 16);
    uint4 x = *at;
    bool bad = false;
    for (uint32_t* w : {&x.x, &x.y, &x.z, &x.w}) {
      const uint32_t m = F == kKvF16 ? __vcmpeq2(*w & 0x7c007c00u, 0x7c007c00u) : __vcmpeq4(*w & 0x7f7f7f7fu, 0x7f7f7f7fu);
      bad |= m != 0;
      *w &= ~m;
    }
    if (bad) *at = x;
    any |= bad;
  }
  umma::fence_proxy_async_smem();
  __syncwarp();  // other lanes read these bytes next (a vote orders no memory)
  return __any_sync(0xffffffffu, any);
}

// ---------------------------------------------------------------- narrow

// Two or four consecutive elements of a query row as f32 (vec: one load).
__device__ __forceinline__ void pair_of_row(const float* p, bool vec, float& a, float& b) {
  if (vec) {
    const float2 x = *reinterpret_cast<const float2*>(p);
    a = x.x; b = x.y;
  } else {
    a = p[0]; b = p[1];
  }
}
__device__ __forceinline__ void pair_of_row(const __half* p, bool vec, float& a, float& b) {
  __half2 x;
  if (vec) x = *reinterpret_cast<const __half2*>(p);
  else x = __halves2half2(p[0], p[1]);
  a = __low2float(x); b = __high2float(x);
}
__device__ __forceinline__ void four_of_row(const float* p, bool vec, float (&v)[4]) {
  if (vec) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[i];
}
__device__ __forceinline__ void four_of_row(const __half* p, bool vec, float (&v)[4]) {
  __half h[4];
  if (vec) *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(p);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = p[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __half2float(h[i]);
}

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
  SeqTables seqs;
};

template <int F, int HD, bool FOLD, typename Q>
__global__ void __launch_bounds__(32 * kWarps, kNarrowCtas)
    narrow_attn_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan p, const __grid_constant__ Maps maps,
                       const int32_t* given, int32_t* cum_out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using N = Narrow<F, HD>;
  using Tl = typename N::Tl;
  constexpr int KEYS = N::kKeys, RT = FOLD ? 8 : 16, kPer = FOLD ? 1 : 2;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ NarrowShared<F, HD> sh;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, tq = lane & 3;
  const int worker = blockIdx.x * kWarps + warp;
  if (t == 0) {
    for (int i = 0; i < kWarps; ++i)
      for (int j = 0; j < N::kStages; ++j) umma::mbar_init(&sh.full[i][j], F == kKvF16 ? 1 : 33);
    sh.abort = 0;
    umma::fence_barrier_init();
  }
  const Seqs cum = sequences(a, p, given, sh.seqs, cum_out);
  __syncthreads();
  uint8_t* tiles = smem + warp * N::kStages * N::kStage;
  float* scales = reinterpret_cast<float*>(smem + kWarps * N::kStages * N::kStage + warp * N::kScales);
  Ahead& ahead = sh.ahead[warp];
  Walk w(p, a, cum, worker);
  if (lane == 0) {
    ahead.w = w;
    ahead.key = ahead.end = 0;
  }
  __syncwarp();
  int issued = 0, done = 0;     // tiles copied and used by this warp: stage = count mod kStages
  // Copy the warp's next tile into the stage whose tile was used last.
  auto copy = [&]() {
    if (ahead.key >= ahead.end) {
      __syncwarp();
      if (lane == 0)
        while (ahead.key >= ahead.end && ahead.w.next(ahead.x, p, a, cum)) {
          ahead.key = ahead.x.t0 * KEYS;
          ahead.end = min(ahead.x.t1 * KEYS, ahead.x.limit);
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
      ahead.key = pos + KEYS;
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

  Rows<F, HD, FOLD, KEYS, sizeof(Q) == 4> st;
  const float base = a.scale * kLog2e;
  Piece x;
  while (w.next(x, p, a, cum)) {
    uint32_t qa[HD / 16][4];
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      // this lane's part of query row g + 8 r: elements 2 tq, 2 tq + 1 (+ 8) of every step's K axis, which are
      // dimensions 4 tq ... of K's words in bytes
      const Q* src = q_row<Q>(a, p, x, g + 8 * r, st.lim[r]);
      float v[HD / 16][4] = {};
      if (src) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          if constexpr (F == kKvF16) {
            pair_of_row(src + 16 * ks + 2 * tq, a.q_vec, v[ks][0], v[ks][1]);
            pair_of_row(src + 16 * ks + 8 + 2 * tq, a.q_vec, v[ks][2], v[ks][3]);
          } else {
            four_of_row(src + 16 * ks + 4 * tq, a.q_vec, v[ks]);
          }
        }
      }
      st.f[r] = base;
      if constexpr (FOLD && sizeof(Q) == 4) {
        uint32_t mx = 0;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = max(mx, __float_as_uint(v[ks][i]) & 0x7fffffffu);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float shrink = row_shrink(mx);
        st.f[r] = base / shrink;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[ks][i] *= shrink;
      }
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          __half2 lead = __floats2half2_rn(v[ks][2 * h], v[ks][2 * h + 1]);
          // K may hold infinities, whose products with a leading part of 0 would be NaN (and with the rest are not looked at)
          if constexpr (FOLD && sizeof(Q) == 4 && F == kKvF16)
            lead = __halves2half2(but_zero(__low2half(lead), v[ks][2 * h]), but_zero(__high2half(lead), v[ks][2 * h + 1]));
          qa[ks][2 * h + r] = half2_bits(lead);
          if constexpr (FOLD) {
            const float2 z = __half22float2(lead);
            qa[ks][2 * h + 1] = half2_bits(__floats2half2_rn(v[ks][2 * h] - z.x, v[ks][2 * h + 1] - z.y));
          }
        }
    }
    st.clear();
    const int end = min(x.t1 * KEYS, x.limit);
    float* part = p.part + x.slot * (RT * HD);
    bool hidden = false, taken = false;
    int steps = 0;
#pragma unroll 1
    for (int key = x.t0 * KEYS; key < end; key += KEYS) {
      if (st.kTake && steps++ == st.kTakeSteps) {
        st.take_out(part + g * HD, 0, taken);
        taken = true;
        steps = 1;
      }
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
      if (F != kKvI8 && key + KEYS > x.fewest && x.fewest < x.limit)
        hidden |= hide_v<F, HD, KEYS>(stage + Tl::kBytes, max(0, x.fewest - key), min(left, KEYS), lane);
      const float* ks = scales + s * (2 * KEYS);
      auto frag = [&](int step, uint32_t (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = qa[step][i];
      };
      if (key + KEYS > x.fewest) st.template step<KEYS / 8, true>(k_base, k_base + Tl::kBytes, ks, ks + KEYS, 0, key, frag);
      else st.template step<KEYS / 8, false>(k_base, k_base + Tl::kBytes, ks, ks + KEYS, 0, key, frag);
      __syncwarp();
      ++done;
    }
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      st.take_out(part + (g + 8 * r) * HD, r, taken);
      const float l = st.denominator(r);
      if (tq == 0) *reinterpret_cast<float2*>(p.ml + 2 * (x.slot * RT + g + 8 * r)) = make_float2(st.m[r], hidden ? -l : l);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // no grid of this call ends before the one it followed
  if (*(volatile int*)&sh.abort) grace();
}

}  // namespace attn
}  // namespace uaii_b200
