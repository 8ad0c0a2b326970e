// attn_wide.cuh -- attention items of many rows on tcgen05 (see prefix_attn.cu).
//
// One CTA per SM works on two row tiles of 128: two softmax warpgroups alternate, so that the tensor core works on one
// tile's products while the other's exponentials are made.
//   rows split   the item's 256 rows are the two tiles, and every key tile serves both (f16 queries, many rows)
//   keys split   the item's 128 rows are both, and each takes every other key tile (f32 queries, whose leading parts and
//                rests are two operands added into one accumulator; or up to 128 rows)
// Per key tile of 64: copied bytes -> (four warps) f16 operands in shared memory, K as [key][dim], V transposed to
// [dim][key] -> S = Q K^T, Q from tensor memory -> (a thread per row) 2^(S - m), weights packed into the tensor memory
// that held S -> O += P V, P from tensor memory.  Q and P in tensor memory leave shared memory's bandwidth to K and V:
// with Q there as well, S alone would read 6 KB per 32 cycles of products.  S and P go by halves of 32 keys: while a
// warpgroup makes one half's weights, the other half's products and the next scores are under way.
// A key tile of 256 f16 rows takes about 3400 cycles, 1930 of them products (the tensor pipe's active half; the weights'
// rests are a third of them): 512 rows a kv head, 8 kv heads, 32801 i8 positions 109 us, 0.63 PFLOP/s of the formula's
// operations, 0.38 of a plain bf16 product's measured rate.  The weights of a half are made by one thread a row at the
// limit of its registers, and do not hide under the other half's products.  A CTA's first scores come after 12000 cycles;
// a further piece costs about seven tiles.  Taking the next piece's queries in before a piece's sums go out was no faster.
// Tensor memory: S and P of tile r, half h at column 64 r + 32 h, Q at 128 + 64 r, O at 256 + 128 r.
#pragma once

#include <type_traits>

#include "attn_common.cuh"

namespace uaii_b200 {
namespace attn {

template <int F, int HD>
struct Wide {
  using Tl = Tile<F, HD, kTile>;
  static constexpr int kRaw = 2 * Tl::kBytes;                       // K, then V
  static constexpr int kRawStages = kRaw > 16384 ? 2 : 3;
  static constexpr int kOpK = kTile * HD * 2, kOp = 2 * kOpK;       // K as [HD / 64][64 keys][128 B], V as [HD][128 B]
  static constexpr int kOps = 4;                                    // operand stages
  static constexpr int kSmem = kOps * kOp + kRawStages * kRaw + 1024;
  static constexpr int kSoft = 256, kConvert = 128, kThreads = kSoft + kConvert + 96;
};

template <int F, int HD>
struct WideShared {
  static constexpr int kRawStages = Wide<F, HD>::kRawStages;
  static constexpr int kOps = Wide<F, HD>::kOps;
  uint64_t raw_full[kRawStages], raw_empty[kRawStages], op_full[kOps], op_empty[kOps];
  uint64_t q_full, q_seen, s_full[2][2], p_full[2][2], o_done[2][2];  // [row tile][half]
  uint32_t tmem;
  int abort;
  alignas(16) float raw_scale[kRawStages][2][kTile];
  alignas(16) float kf[kOps][kTile];   // K scale * softmax scale * log2(e)
  alignas(16) float vf[kOps][kTile];   // V scale
  alignas(16) float vlog[kOps][kTile]; // its log2_scale
  float vmost[kOps];                   // the largest of a tile, at least kLeastScale
  alignas(4) uint8_t hidden[kOps][4];  // by the converting warps: V values that not all rows see were left out
  SeqTables seqs;
};

__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

__device__ __forceinline__ int tiles_of(const Piece& x) { return min(x.t1, (x.limit + kTile - 1) / kTile) - x.t0; }

// ---------------------------------------------------------------- copies

template <int F, int HD>
__device__ void wide_copy(const PrefixAttnArgs& a, const Plan& p, const Maps& maps, const Seqs& seqs, uint8_t* raw,
                          WideShared<F, HD>& sh) {
  using Wd = Wide<F, HD>;
  using Tl = typename Wd::Tl;
  const int lane = threadIdx.x & 31;
  Walk w(p, a, seqs, blockIdx.x);
  Piece x;
  int count = 0;
  while (w.next(x, p, a, seqs)) {
    const KvCache& c = x.own ? a.own : a.prefix;
    const CUtensorMap *mk = x.own ? &maps.ok : &maps.pk, *mv = x.own ? &maps.ov : &maps.pv;
    for (int i = 0, n = tiles_of(x); i < n; ++i, ++count) {
      const int s = count % Wd::kRawStages, pos = (x.t0 + i) * kTile;
      umma::bounded_wait(&sh.raw_empty[s], ((count / Wd::kRawStages) & 1) ^ 1, &sh.abort, a.err, kErrKvCopy);
      if (*(volatile int*)&sh.abort) return;
      uint64_t* bar = &sh.raw_full[s];
      if (lane == 0) {
        umma::mbar_arrive_expect_tx(bar, 2 * Tl::kBytes);
        const uint32_t dst = umma::smem_u32(raw + s * Wd::kRaw);
#pragma unroll
        for (int b = 0; b < Tl::kBoxes; ++b) {
          tma_load_3d(dst + b * Tl::kBoxBytes, mk, bar, b * (Tl::kPart / Tl::kEsz), pos, x.z);
          tma_load_3d(dst + Tl::kBytes + b * Tl::kBoxBytes, mv, bar, b * (Tl::kPart / Tl::kEsz), pos, x.z);
        }
      }
      if constexpr (F != kKvF16) {  // row scales: 4-byte copies, zero past the end of the cache
#pragma unroll
        for (int j = 0; j < 2 * kTile / 32; ++j) {
          const int k = (j % (kTile / 32)) * 32 + lane;
          const bool in = pos + k < c.max_seq;
          const float* src = (j < kTile / 32 ? c.k_scale : c.v_scale) + (int64_t)x.z * c.max_seq + (in ? pos + k : 0);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(umma::smem_u32(&sh.raw_scale[s][0][0]) + (j * 32 + lane) * 4),
                       "l"(src), "r"(in ? 4 : 0)
                       : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(umma::smem_u32(bar)) : "memory");
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------- bytes to operands

template <int F, int HD>
__device__ void wide_convert(const PrefixAttnArgs& a, const Plan& p, const Seqs& seqs, uint8_t* ops, uint8_t* raw,
                             WideShared<F, HD>& sh) {
  using Wd = Wide<F, HD>;
  using Tl = typename Wd::Tl;
  constexpr int kPieces = Tl::kRow / 16;
  const int lane = threadIdx.x & 31, cw = ((int)threadIdx.x - Wd::kSoft) >> 5;  // keys 16 cw .. 16 cw + 15
  const int mi = lane >> 3, r8 = lane & 7, tq = lane & 3;
  const float base = a.scale * kLog2e;
  Walk w(p, a, seqs, blockIdx.x);
  Piece x;
  int count = 0;
  while (w.next(x, p, a, seqs)) {
    for (int i = 0, n = tiles_of(x); i < n; ++i, ++count) {
      const int s = count % Wd::kRawStages, o = count % Wd::kOps, left = x.limit - (x.t0 + i) * kTile;
      umma::bounded_wait(&sh.raw_full[s], (count / Wd::kRawStages) & 1, &sh.abort, a.err, kErrKvCopy);
      umma::bounded_wait(&sh.op_empty[o], ((count / Wd::kOps) & 1) ^ 1, &sh.abort, a.err, kErrKvCopy);
      const uint32_t rk = umma::smem_u32(raw + s * Wd::kRaw), rv = rk + Tl::kBytes;
      const uint32_t ok = umma::smem_u32(ops + o * Wd::kOp), ov = ok + Wd::kOpK;
      // K: 16-byte chunk c of an operand row holds positions 8 c ... of the MMA's K axis; chunks of 64 dimensions apart
      // lie 8 KB apart
      auto k_to = [&](int row, int c) { return ok + (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4); };
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int row = 16 * cw + 8 * g + r8;
#pragma unroll
        for (int c = 0; c < kPieces; c += 4) {
          uint32_t v[4];
          ldsm4(v, piece<F, HD, kTile>(rk, row, c + mi));
          if constexpr (F == kKvF16) {
            stsm4(k_to(row, c + mi), v[0], v[1], v[2], v[3]);
          } else {  // a word's four dimensions go to chunks 2 c and 2 c + 1 (operand_dim)
            uint32_t b[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) unpack<F, false>(v[j], b[2 * j], b[2 * j + 1]);
            stsm4(k_to(row, 2 * c + mi), b[0], b[1], b[2], b[3]);
            stsm4(k_to(row, 2 * c + 4 + mi), b[4], b[5], b[6], b[7]);
          }
        }
      }
      // V transposed: 8-bit pieces hold 16 dimensions, whose even ones become rows 16 c .. 16 c + 7 and odd ones the next
      // eight.  Nothing is stored past the item's last position: zeros, since 0 * NaN would not be 0.  Nor may an infinity
      // or a NaN that only some of the item's tokens see meet the zero weights of the others: a zero instead, and the
      // joining kernel gives it to those that see it.
      auto v_to = [&](int row) { return ov + row * 128 + (((2 * cw + (mi & 1)) ^ (row & 7)) << 4); };
      const int all_see = x.fewest < x.limit ? x.fewest - (x.t0 + i) * kTile : left;
      const bool end = F != kKvI8 && all_see < kTile;
      bool hidden = false;
      auto keep = [&](uint32_t pair, int key) {
        pair &= key + 1 < left ? ~0u : key < left ? 0xffffu : 0u;
        uint32_t m = __vcmpeq2(pair & 0x7c007c00u, 0x7c007c00u);
        m &= key >= all_see ? ~0u : key + 1 >= all_see ? ~0xffffu : 0u;
        hidden |= m != 0;
        return pair & ~m;
      };
#pragma unroll
      for (int c = 0; c < kPieces; c += 2) {
        uint32_t v[4];
        ldsm4t(v, piece<F, HD, kTile>(rv, 16 * cw + 8 * (mi & 1) + r8, c + (mi >> 1)));
        const int lo = 16 * cw + 2 * tq, hi = lo + 8;
        if constexpr (F == kKvF16) {
          if (end) {
            v[0] = keep(v[0], lo); v[1] = keep(v[1], hi);
            v[2] = keep(v[2], lo); v[3] = keep(v[3], hi);
          }
          stsm4(v_to(8 * (c + (mi >> 1)) + r8), v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t e0, d0, e1, d1;
            unpack<F, true>(v[2 * j], e0, d0);
            unpack<F, true>(v[2 * j + 1], e1, d1);
            if (end) {
              e0 = keep(e0, lo); d0 = keep(d0, lo);
              e1 = keep(e1, hi); d1 = keep(d1, hi);
            }
            stsm4(v_to(16 * (c + j) + 8 * (mi >> 1) + r8), e0, e1, d0, d1);
          }
        }
      }
      if constexpr (F != kKvF16) {
        if (cw == 0) {  // the tile's column factors
          float most = kLeastScale;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int k = 32 * j + lane;
            const float vx = k < left ? sh.raw_scale[s][1][k] : 0.f;  // nothing is stored past the last position
            sh.kf[o][k] = sh.raw_scale[s][0][k] * base;
            sh.vf[o][k] = vx;
            sh.vlog[o][k] = log2_scale(vx);
            most = fmaxf(most, fabsf(vx));  // (a NaN shows in its products, not here)
          }
          const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
          if (lane == 0) sh.vmost[o] = __uint_as_float(top);
        }
      }
      if constexpr (F != kKvI8) hidden = __any_sync(0xffffffffu, hidden);
      umma::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if constexpr (F != kKvI8) sh.hidden[o][cw] = hidden;
        umma::mbar_arrive(&sh.raw_empty[s]);
        umma::mbar_arrive(&sh.op_full[o]);
      }
    }
  }
}

// ---------------------------------------------------------------- products

// The tensor cores cut sums off where they should round (a loss of 1.5e-8 of an f32 sum at each of its additions, 8 a
// key tile of f32 queries: 5e-6 in 46 tiles), so f32 sums are taken out after this many tiles and added up in f32.
constexpr int kDrain = 5;

// One warp per row tile r: the scores of a half, then, when its weights are there, O += P V; when those products are
// done, the half of the next key tile takes P's place.  The whole warp stays together and one lane issues: the descriptors
// then live in uniform registers.
template <int F, int HD, bool SPLIT_Q>
__device__ void wide_products(const PrefixAttnArgs& a, const Plan& p, const Seqs& seqs, uint8_t* ops, WideShared<F, HD>& sh,
                              int r) {
  using Wd = Wide<F, HD>;
  constexpr uint32_t kIdS = umma::idesc_f16_f32(128, kTile / 2), kIdO = umma::idesc_f16_f32(128, HD);
  const uint32_t tm = sh.tmem, ts = tm + 64 * r, to = tm + 256 + 128 * r;
  const uint32_t q = tm + 128 + (p.split_keys ? 0 : 64 * r);
  Walk w(p, a, seqs, blockIdx.x);
  Piece x;
  int count = 0, pieces = 0;
  uint32_t mine = 0;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    umma::bounded_wait(bar, parity, &sh.abort, a.err, kErrKvCopy);
    umma::tc_fence_after();
  };
  auto operand = [&](int o) { return umma::sw128_desc(umma::smem_u32(ops + o * Wd::kOp)); };
  auto scores = [&](int o, int h) {  // 32 rows (4 KB) of K; 32 bytes a step, 64 dimensions a swizzled block
    const uint64_t k = operand(o) + (uint64_t)(h * (32 * 128) >> 4);
    if (umma::elect_one()) {
      // the rests first: every addition cuts the running sum off, and theirs is small
#pragma unroll
      for (int part = SPLIT_Q; part >= 0; --part)
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
          umma::mma_f16_ts(ts + 32 * h, q + 64 * part + 8 * ks, k + (uint64_t)(((ks >> 2) * (kTile * 128) + (ks & 3) * 32) >> 4),
                           kIdS, part != SPLIT_Q || ks);
      umma::mma_commit(&sh.s_full[r][h]);
    }
    __syncwarp();
  };
  while (w.next(x, p, a, seqs)) {
    const int n = tiles_of(x), first = p.split_keys ? r : 0, step = p.split_keys ? 2 : 1;
    if (n <= 0) continue;
    int summed = 0;
    wait(&sh.q_full, pieces++ & 1);
    if (umma::elect_one()) umma::mbar_arrive(&sh.q_seen);
    __syncwarp();
    if (first < n) {
      const int o = (count + first) % Wd::kOps;
      wait(&sh.op_full[o], ((count + first) / Wd::kOps) & 1);
      scores(o, 0);
      scores(o, 1);
    }
    for (int i = first; i < n; i += step, ++mine, ++summed) {
      if (SPLIT_Q && summed == kDrain) summed = 0;  // (the sums are taken out, by then)
      const int o = (count + i) % Wd::kOps, on = (count + i + step) % Wd::kOps;
      const uint64_t v = operand(o) + (Wd::kOpK >> 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wait(&sh.p_full[r][h], mine & 1);
        if (umma::elect_one()) {
#pragma unroll
          for (int part = 0; part < 2; ++part)  // leading parts of the weights, then the rests
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
              umma::mma_f16_ts(to, ts + 32 * h + 16 * part + 8 * ks, v + 2 * (2 * h + ks), kIdO, summed || h || part || ks);
          umma::mma_commit(&sh.o_done[r][h]);
          if (h) umma::mma_commit(&sh.op_empty[o]);
        }
        __syncwarp();
        if (i + step < n) {
          if (h == 0) wait(&sh.op_full[on], ((count + i + step) / Wd::kOps) & 1);
          wait(&sh.o_done[r][h], mine & 1);
          scores(on, h);
        }
      }
    }
    count += n;
  }
}

// ---------------------------------------------------------------- softmax

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Two f32 operations in one instruction (each rounded as usual).
__device__ __forceinline__ uint64_t pair_bits(float2 a) { return ((uint64_t)__float_as_uint(a.y) << 32) | __float_as_uint(a.x); }
__device__ __forceinline__ float2 pair_of(uint64_t v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return pair_of(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(d);
}

constexpr int kHalf = kTile / 2;  // keys of a half

// The largest sum of a half's weights, times the tile's largest V scale, for which every product is surely an f16.  (At or
// below the reference products are at most 2^9.)
constexpr float kMostSum = 46000.f;

// Operand position -> dimension: K's words hold four consecutive dimensions of a byte row, which lie in two chunks of an
// operand row.  Even positions keep their neighbour.
template <int F>
__device__ __forceinline__ int operand_dim(int pos) {
  if constexpr (F == kKvF16) return pos;
  return (pos & ~15) | ((pos & 6) << 1) | ((pos & 8) >> 2) | (pos & 1);
}

// This thread's row of q (null: zeros) into tensor memory as operand `part` (1: the rests of a split); returns the power
// of two by which a split row was multiplied.
template <int F, int HD, bool SPLIT_Q, typename Q>
__device__ __forceinline__ float put_q(const Q* src, bool vec, int part, uint32_t taddr) {
  float shrink = 1.f;
  constexpr int kVec = 16 / sizeof(Q), kLoads = 64 / kVec;
  union Block {
    uint4 u[kLoads];
    Q e[64];
  };
  auto load = [&](int h, Block& v) {  // dimensions 64 h ..., every load under way before the first is used
    if (src == nullptr) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) v.u[i] = make_uint4(0, 0, 0, 0);
    } else if (vec) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) v.u[i] = reinterpret_cast<const uint4*>(src + 64 * h)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 64; ++i) v.e[i] = src[64 * h + i];
    }
  };
  if constexpr (SPLIT_Q) {
    uint32_t mx = 0;
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) {
      Block v;
      load(h, v);
#pragma unroll
      for (int i = 0; i < 64; ++i) mx = max(mx, __float_as_uint((float)v.e[i]) & 0x7fffffffu);
    }
    shrink = row_shrink(mx);
  }
  Block all[SPLIT_Q ? 1 : HD / 64];  // (f32 rows are too long to hold whole)
  if constexpr (!SPLIT_Q)
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) load(h, all[h]);
#pragma unroll
  for (int h = 0; h < HD / 64; ++h) {
    Block& v = all[SPLIT_Q ? 0 : h];
    if constexpr (SPLIT_Q) load(h, v);
    uint32_t c[32];
    if constexpr (!SPLIT_Q) {  // pairs as they are
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const int d = operand_dim<F>(2 * j) / 2;
        const uint4 x = v.u[d >> 2];
        c[j] = (d & 3) == 0 ? x.x : (d & 3) == 1 ? x.y : (d & 3) == 2 ? x.z : x.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const int d = operand_dim<F>(2 * j);
        const float y0 = (float)v.e[d] * shrink, y1 = (float)v.e[d + 1] * shrink;
        __half2 e = __floats2half2_rn(y0, y1);
        if constexpr (F == kKvF16) {
          // K may hold infinities: both parts have the value's sign, and neither is 0 (their products would be NaN)
          // unless the value is.  With the leading part rounded towards zero the rest leaves 2^-22 of the largest.
          e = __halves2half2(but_zero(__float2half_rz(y0), y0), but_zero(__float2half_rz(y1), y1));
          if (part) {
            const float2 z = __half22float2(e);
            auto rest = [](float y, float z) {  // (a leading part that is larger than its value was made of 0)
              return but_zero(__float2half_rn(fabsf(z) > fabsf(y) ? 0.f : y - z), y);
            };
            e = __halves2half2(rest(y0, z.x), rest(y1, z.y));
          }
        } else if (part) {
          const float2 z = __half22float2(e);
          e = __floats2half2_rn(y0 - z.x, y1 - z.y);
        }
        c[j] = half2_bits(e);
      }
    }
    umma::tmem_st32(taddr + 32 * h, c);
  }
  umma::tmem_st_wait();
  return shrink;
}

// 32 bytes, a whole sector: a thread's row lies apart from its neighbours'.
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

template <int F, int HD, bool SPLIT_Q, typename Q>
__device__ void wide_softmax(const PrefixAttnArgs& a, const Plan& p, const Seqs& seqs, WideShared<F, HD>& sh) {
  const int lane = threadIdx.x & 31, warp = (int)threadIdx.x >> 5, r = warp >> 2, row = threadIdx.x & 127;
  const uint32_t tm = sh.tmem + ((uint32_t)(32 * (warp & 3)) << 16);  // this warp's 32 lanes of tensor memory
  const uint32_t ts = tm + 64 * r, to = tm + 256 + 128 * r;
  const float base = a.scale * kLog2e;
  Walk w(p, a, seqs, blockIdx.x);
  Piece x;
  int count = 0;            // key tiles of the CTA
  uint32_t mine = 0;        // key tiles of this warpgroup
  int pieces = 0;           // with keys
  while (w.next(x, p, a, seqs)) {
    const int n = tiles_of(x), step = p.split_keys ? 2 : 1, first = p.split_keys ? r : 0;
    int lim;
    const Q* src = q_row<Q>(a, p, x, p.split_keys ? row : 128 * r + row, lim);
    float m = -INFINITY, l = 0.f, row_f = 1.f;
    uint32_t hidden = 0;
    const int64_t at_row = x.slot * 256 + 128 * r + row;
    float* part = p.part + at_row * HD;
    int summed = 0;           // key tiles in the sums that tensor memory holds
    float drained_m = 0.f;    // the reference of the sums taken out before
    bool drained = false;
    // The sums so far to the workspace, added to those taken out before.
    auto drain = [&]() {
      umma::bounded_wait(&sh.o_done[r][1], (mine - 1) & 1, &sh.abort, a.err, kErrKvCopy);
      umma::tc_fence_after();
      const float old = drained_m == m ? 1.f : ex2(drained_m - m);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t u[32];
        tmem_ld32(to + 32 * c, u);
        umma::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          // 8-bit pieces: even dimensions of 16 lie before the odd ones
          float z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) z[i] = __uint_as_float(u[F == kKvF16 ? j + i : (j & 16) + ((j & 15) >> 1) + (i >> 1) + 8 * (i & 1)]);
          if (SPLIT_Q && drained) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 v = *reinterpret_cast<const float4*>(part + 32 * c + j + i);
              z[i] = fmaf(v.x, old, z[i]);
              z[i + 1] = fmaf(v.y, old, z[i + 1]);
              z[i + 2] = fmaf(v.z, old, z[i + 2]);
              z[i + 3] = fmaf(v.w, old, z[i + 3]);
            }
          }
          store8(part + 32 * c + j, z);
        }
      }
      umma::tc_fence_before();
      drained = true;
      drained_m = m;
    };
    if (n > 0) {
      // Both issuing warps have seen the piece before's queries: with one tile and split keys the second has nothing to
      // issue, and nothing else would keep the barrier's phase from passing it by.
      if (pieces++) umma::bounded_wait(&sh.q_seen, pieces & 1, &sh.abort, a.err, kErrKvCopy);
      if (p.split_keys) asm volatile("bar.sync 1, 256;" ::: "memory");  // the other half's products with q are done
      const float shrink = put_q<F, HD, SPLIT_Q, Q>(src, a.q_vec, r, tm + 128 + 64 * r);
      if constexpr (SPLIT_Q) row_f = 1.f / shrink;
      umma::tc_fence_before();
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(&sh.q_full);
    }
    for (int i = first; i < n; i += step, ++mine, ++summed) {
      if (SPLIT_Q && summed == kDrain) {
        drain();
        summed = 0;
      }
      const int at = count + i, o = at % Wide<F, HD>::kOps;
      umma::bounded_wait(&sh.op_full[o], (at / Wide<F, HD>::kOps) & 1, &sh.abort, a.err, kErrKvCopy);  // the column factors
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const int pos0 = (x.t0 + i) * kTile + kHalf * h;
        const uint32_t tsh = ts + kHalf * h;
        umma::bounded_wait(&sh.s_full[r][h], mine & 1, &sh.abort, a.err, kErrKvCopy);
        umma::tc_fence_after();
        float s[kHalf];
        auto load = [&]() {
          tmem_ld32(tsh, reinterpret_cast<uint32_t*>(s));
          umma::tmem_ld_wait();
        };
        load();
        const bool masked = pos0 + kHalf > x.fewest;
        const int seen = masked ? lim - pos0 : kHalf;
        const float *kf = &sh.kf[o][kHalf * h], *vf = &sh.vf[o][kHalf * h];
        // Weights against the reference as it is, and the operand made of them; their sum tells whether one is too
        // large.  No maximum is made then.  (cut: columns from `seen` on get no weight, whatever their scale is.)
        uint32_t pk[kHalf / 2], rests[kHalf / 2];
        auto weights = [&](auto cut) {
          const float off = kLift - (m == -INFINITY ? 0.f : m);
          float2 sum[2] = {};
#pragma unroll
          for (int j = 0; j < kHalf; j += 4) {
            float4 f = make_float4(base, base, base, base), v = make_float4(1.f, 1.f, 1.f, 1.f);
            if constexpr (F != kKvF16) {
              f = *reinterpret_cast<const float4*>(kf + j);
              v = *reinterpret_cast<const float4*>(vf + j);
            }
            if constexpr (SPLIT_Q) f = make_float4(f.x * row_f, f.y * row_f, f.z * row_f, f.w * row_f);
            float2 w[2] = {fma2(make_float2(s[j], s[j + 1]), make_float2(f.x, f.y), make_float2(off, off)),
                           fma2(make_float2(s[j + 2], s[j + 3]), make_float2(f.z, f.w), make_float2(off, off))};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              w[k] = make_float2(ex2(w[k].x), ex2(w[k].y));
              if constexpr (cut.value) {
                if (j + 2 * k >= seen) w[k].x = 0.f;
                if (j + 2 * k + 1 >= seen) w[k].y = 0.f;
              }
              sum[k] = add2(sum[k], w[k]);
              if constexpr (F != kKvF16) {
                w[k] = mul2(w[k], k ? make_float2(v.z, v.w) : make_float2(v.x, v.y));
                if constexpr (cut.value) {
                  if (j + 2 * k >= seen) w[k].x = 0.f;
                  if (j + 2 * k + 1 >= seen) w[k].y = 0.f;
                }
              }
              split_weights<F == kKvF16>(w[k].x, w[k].y, pk[j / 2 + k], rests[j / 2 + k]);
            }
          }
          return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        };
        float sum = 0.f, vmost = 1.f;
        if constexpr (F != kKvF16) vmost = sh.vmost[o];
        bool slow = __any_sync(0xffffffffu, masked || m == -INFINITY);
        if (!slow) {
          sum = weights(std::false_type{});
          slow = __any_sync(0xffffffffu, !(sum * vmost <= kMostSum));
          if (slow) load();  // S is still in tensor memory
        }
        if (slow) {
          if constexpr (F != kKvI8) hidden |= *reinterpret_cast<const uint32_t*>(sh.hidden[o]);
          float top = -INFINITY, product = -INFINITY, shrink_o = 1.f;
#pragma unroll
          for (int j = 0; j < kHalf; ++j) {
            if (j >= seen) continue;
            const float y = s[j] * ((F == kKvF16 ? base : kf[j]) * row_f);
            top = fmaxf(top, y);
            if constexpr (F != kKvF16) product = fmaxf(product, y + sh.vlog[o][kHalf * h + j]);
          }
          const float next = next_reference(m, top, F == kKvF16 ? top : product);
          if (next > m + (m == -INFINITY ? 0.f : kSlack)) {
            shrink_o = ex2(m - next);
            l *= shrink_o;
            m = next;
          }
          if ((h || summed) && __any_sync(0xffffffffu, shrink_o != 1.f)) {
            // the products made so far, up to those of the half before, rest
            umma::bounded_wait(&sh.o_done[r][h ^ 1], (h ? mine : mine - 1) & 1, &sh.abort, a.err, kErrKvCopy);
            umma::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t y[16];
              umma::tmem_ld16(to + 16 * c, y);
              umma::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * shrink_o);
              tmem_st16(to + 16 * c, y);
            }
          }
          sum = weights(std::true_type{});
        }
        l += sum;
        tmem_st16(tsh, pk);
        tmem_st16(tsh + kHalf / 2, rests);
        umma::tmem_st_wait();
        umma::tc_fence_before();
        __syncwarp();
        if (lane == 0) umma::mbar_arrive(&sh.p_full[r][h]);
      }
    }
    count += n > 0 ? n : 0;
    *reinterpret_cast<float2*>(p.ml + 2 * at_row) = make_float2(m, hidden ? -l : l);
    if (n > first) {
      drain();
    } else {
#pragma unroll 4
      for (int j = 0; j < HD; j += 4) reinterpret_cast<float4*>(part + j)[0] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    umma::tc_fence_before();
  }
}

template <int F, int HD, typename Q>
__global__ void __launch_bounds__(Wide<F, HD>::kThreads, 1)
    wide_attn_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan p, const __grid_constant__ Maps maps,
                     const int32_t* given, int32_t* cum_out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // they take the SMs over as this grid leaves them
  using Wd = Wide<F, HD>;
  constexpr bool kSplitQ = sizeof(Q) == 4;
  extern __shared__ uint8_t dynamic[];
  uint8_t* ops = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dynamic) + 1023) & ~uintptr_t(1023));
  uint8_t* raw = ops + Wd::kOps * Wd::kOp;
  __shared__ WideShared<F, HD> sh;
  const int t = threadIdx.x, warp = t >> 5;
  constexpr int kCopyWarp = (Wd::kSoft + Wd::kConvert) / 32, kProductWarp = kCopyWarp + 1;
  if (t == 0) {
    for (int i = 0; i < Wd::kRawStages; ++i) {
      umma::mbar_init(&sh.raw_full[i], F == kKvF16 ? 1 : 33);
      umma::mbar_init(&sh.raw_empty[i], Wd::kConvert / 32);
    }
    for (int i = 0; i < Wd::kOps; ++i) {
      umma::mbar_init(&sh.op_full[i], Wd::kConvert / 32);
      umma::mbar_init(&sh.op_empty[i], p.split_keys ? 1 : 2);
    }
    for (int i = 0; i < 2; ++i) {
      for (int h = 0; h < 2; ++h) {
        umma::mbar_init(&sh.s_full[i][h], 1);
        umma::mbar_init(&sh.p_full[i][h], 4);
        umma::mbar_init(&sh.o_done[i][h], 1);
      }
    }
    umma::mbar_init(&sh.q_full, 8);
    umma::mbar_init(&sh.q_seen, 2);
    sh.abort = 0;
    umma::fence_barrier_init();
  }
  if (warp == kProductWarp) umma::tmem_alloc(&sh.tmem, 512);
  const Seqs seqs = sequences(a, p, given, sh.seqs, cum_out);
  umma::tc_fence_before();
  __syncthreads();
  umma::tc_fence_after();
  if (t < Wd::kSoft) wide_softmax<F, HD, kSplitQ, Q>(a, p, seqs, sh);
  else if (t < Wd::kSoft + Wd::kConvert) wide_convert<F, HD>(a, p, seqs, ops, raw, sh);
  else if (warp == kCopyWarp) wide_copy<F, HD>(a, p, maps, seqs, raw, sh);
  else wide_products<F, HD, kSplitQ>(a, p, seqs, ops, sh, warp - kProductWarp);
  __syncwarp();
  if (*(volatile int*)&sh.abort) grace();
  umma::tc_fence_before();
  __syncthreads();
  if (warp == kProductWarp) umma::tmem_dealloc(sh.tmem, 512);
}

}  // namespace attn
}  // namespace uaii_b200
