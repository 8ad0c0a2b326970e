// prefix_attn.cu -- attention of new tokens over a prefix that the whole batch shares and each sequence's own
// cached positions, straight from an f16 or 8-bit cache (formats: kv_cache.cu).
//
//   s_j = scale * ks_j * (q . c_j),   out = sum_j e^(s_j - m) vs_j c'_j / sum_j e^(s_j - m)
//
// with c_j, c'_j the stored K and V values of position j and ks_j, vs_j their row scales (1 for f16).
// Token t of sequence b sees prefix positions [0, P) and own positions [0, own_len[b] - T + t]; a row that sees
// none is zero.  References, sums and outputs are f32.
//
// Work.  An item is a tile of query rows that read the same keys: (kv head, rows of the whole batch) over the
// prefix, (sequence, kv head, rows) over own positions.  Its keys come in units, a few more of them in front of each
// item for what a piece costs besides; the units of all items, laid end to end, are dealt out evenly to the workers (CTAs
// or warps), so a share starts and ends inside items.  Every piece of an item leaves its unnormalised sums, references and
// denominators in the workspace (slot = item + worker, unique because each next piece raises one of the two), and a last
// kernel joins the pieces of each row in a fixed order.
//
// Two tilings, one kernel each.  Bytes become exact f16 operands (the row scales act on scores and probabilities);
// accumulators are f32.
//   narrow  (attn_narrow.cuh) 8 or 16 rows; every warp takes other keys, from copies of its own (few rows: the keys are
//           the work).
//   wide    (attn_wide.cuh) 128 or 256 rows on tcgen05, operands made once for all rows (many rows: the products and the
//           exponentials are the work).
// f32 queries are split in two f16 parts, and so are the weights of all queries: rows 0-7 of an MMA hold the leading parts
// and rows 8-15 the rests ("folded"), which keeps f32 accuracy at no cost while an item has no more than 8 rows; items of
// more rows add a second product with the rests.  Weights of f16 queries in one part cost less (128 sequences behind 32801
// positions 117.6 against 132.8 us, 64 behind 8192 47.4 against 49.3, items of 16 rows 70 against 78) but a result's error
// was 2.9e-4 where its own rounding to f16 makes 2.1e-4, and which of the two a call got went by its rows.
#include <algorithm>

#include "attn_narrow.cuh"
#include "attn_wide.cuh"

namespace uaii_b200 {
namespace attn {
namespace {

// The tables of batches too large for a CTA's shared memory: cum [B + 1], then len [B].
__global__ void __launch_bounds__(1024) sequences_kernel(const __grid_constant__ PrefixAttnArgs a, int unit, int lead, int32_t* cum) {
  __shared__ int warp_sum[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int before = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += 1024) {
    const int64_t b = b0 + t;
    const int len = b < a.B ? own_length(a, b, true) : 0, n = scan32(b < a.B ? units_of(len, unit, lead) : 0);
    if (lane == 31) warp_sum[warp] = n;
    __syncthreads();
    const int s = warp_sum[lane], up_to = __reduce_add_sync(0xffffffffu, lane < warp ? s : 0);
    if (b < a.B) {
      cum[b + 1] = before + up_to + n;
      cum[a.B + 1 + b] = len;
    }
    before += __reduce_add_sync(0xffffffffu, s);
    __syncthreads();
  }
  if (t == 0) cum[0] = 0;
}

// Where one row's pieces lie: n of them, piece k's row at `first` + k * stride (+ odd * sub where an item has two parts).
struct Pieces {
  const float* part;
  const float* ml;
  int64_t first;
  int n, stride, odd, sub;
  __device__ __forceinline__ int64_t row(int k) const { return first + (int64_t)(k >> odd) * stride + (k & odd) * sub; }
};

template <bool OWN>
__device__ __forceinline__ Pieces pieces_of(const PrefixAttnArgs& a, const Plan& p, const int32_t* cum, int b, int rho, int kvh) {
  Pieces q{};
  if (!OWN && p.prefix_items == 0) return q;
  const int j = rho / p.by_rt, per = (int)a.own.heads * p.own_nrt, prefix = p.prefix_items * p.prefix_units;
  const int total = prefix + (per ? cum[a.B] * per : 0);
  int64_t item;
  int u0, units;
  if (OWN) {
    const int before = cum[b];
    units = cum[b + 1] - before;
    item = (int64_t)p.prefix_items + (int64_t)b * per + kvh * p.own_nrt + j;
    u0 = prefix + before * per + (kvh * p.own_nrt + j) * units;
  } else {
    units = p.prefix_units;
    item = kvh * p.prefix_nrt + j;
    u0 = (int)item * units;
  }
  if (units == 0) return q;
  const int each = total / p.by_workers;
  const int c0 = share_of(u0 + p.lead, total, p.workers, each), c1 = share_of(u0 + units - 1, total, p.workers, each);
  q.part = p.part;
  q.ml = p.ml;
  q.first = (item + c0) * p.slot_rows + (rho - j * p.rt);
  q.n = (c1 - c0 + 1) * p.subs;
  q.stride = p.slot_rows;
  q.odd = p.subs - 1;
  q.sub = p.rt;
  return q;
}

// out = sum over a row's pieces of 2^(m - M) o / sum of 2^(m - M) l.  WARPS warps per row; the pieces are taken in the
// order of the workers, prefix first, a warp every WARPS-th.  Bound by latency (lengths, then maxima, then sums: 4 to 8 us
// whatever the rows); inside the narrow kernel, by the worker that comes last, it cost more (6 % of a call of 64
// sequences behind 8192 positions).  px, po: the plans of the kernels that took the prefix and
// the own items.  cum is not __restrict__: it is written while this grid waits, and a load of data declared unchanging may
// be moved in front of the wait.
template <int HD, typename Q, int WARPS>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ Plan px,
                                                   const __grid_constant__ Plan po, const int32_t* cum) {
  constexpr int N = HD / 32, kRows = 4 / WARPS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wr = warp % WARPS;
  const int rows = (int)(a.B * a.T * a.H), row = (int)blockIdx.x * kRows + warp / WARPS;
  const bool live = row < rows;
  const int bt = live ? row / (int)a.H : 0, h = live ? row - bt * (int)a.H : 0, b = bt / (int)a.T, t = bt - b * (int)a.T;
  const int kvh = h / po.by_G, g = h - kvh * po.G;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the pieces are there from here on
  const Pieces qp = pieces_of<false>(a, px, cum, b, bt * po.G + g, kvh), qo = pieces_of<true>(a, po, cum, b, t * po.G + g, kvh);
  // the row's reference, a piece a lane
  float mx = -INFINITY;
  for (int k = lane; k < qp.n; k += 32) mx = fmaxf(mx, qp.ml[2 * qp.row(k)]);
  for (int k = lane; k < qo.n; k += 32) mx = fmaxf(mx, qo.ml[2 * qo.row(k)]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  const float safe = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, o[N] = {};
  bool hidden = false;  // the sign of a piece's l: it left out infinities or NaNs of V
  auto add = [&](const Pieces& s) {
#pragma unroll 4
    for (int k = wr; k < s.n; k += WARPS) {
      const int64_t r = s.row(k);
      const float2 ml = *reinterpret_cast<const float2*>(s.ml + 2 * r);
      float y[N];
      if constexpr (N == 4) *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(s.part + r * HD + N * lane);
      else *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(s.part + r * HD + N * lane);
      const float f = ex2(ml.x - safe);
      l = fmaf(f, fabsf(ml.y), l);
      hidden |= signbit(ml.y);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(f, y[i], o[i]);
    }
  };
  add(qp);
  add(qo);
  if constexpr (WARPS > 1) {
    __shared__ float all[WARPS][HD + 1];
#pragma unroll
    for (int i = 0; i < N; ++i) all[wr][N * lane + i] = o[i];
    if (lane == 0) all[wr][HD] = l;
    hidden = __syncthreads_or(hidden);
    if (wr != 0) return;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
      l += all[w][HD];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] += all[w][N * lane + i];
    }
  }
  if (!live) return;
  if (hidden) {  // positions that the item's first token does not see and this one does
    const int seen = own_length(a, b, false) - (int)a.T + 1, first = (t * po.G + g) / po.by_rt * po.rt / po.by_G;
    const int64_t plane = ((int64_t)b * a.own.heads + kvh) * a.own.max_seq;
    for (int pos = max(0, seen + first); pos < seen + t; ++pos) {
      const int64_t at = (plane + pos) * HD + N * lane;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float v;
        if (a.own.fmt == kKvF16) v = __half2float(static_cast<const __half*>(a.own.v)[at + i]);
        else v = (static_cast<const uint8_t*>(a.own.v)[at + i] & 0x7f) == 0x7f ? NAN : 0.f;
        if (!isfinite(v)) o[i] += v;
      }
    }
  }
  Q y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = (Q)(l == 0.f ? 0.f : __fdiv_rn(o[i], l));
  Q* out = static_cast<Q*>(a.out) + (int64_t)row * HD + N * lane;
  if constexpr (sizeof(y) == 16) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(y);
  else if constexpr (sizeof(y) == 8) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
  else *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(y);
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

constexpr int kWideLead = 7, kNarrowLead = 2;

// The grids of a call and the workspace.  Own items of more than 16 rows: one wide grid for them and the prefix.  Else a
// grid for the prefix (wide above 16 rows) and a narrow one for the own items.
struct Layout {
  Plan prefix, own;        // prefix.grid 0: none, or own's grid takes the prefix too
  bool prefix_wide = false, own_wide = false;
  size_t bytes = 0;
  int64_t most = 0;        // units of a grid, at most
  const Plan& of_prefix() const { return prefix.grid ? prefix : own; }
};

Layout lay_out(const PrefixAttnArgs& a, char* ws) {
  Layout l{};
  const int G = (int)(a.H / a.own.heads), own_rows = (int)(a.T * G), prefix_rows = (int)(a.B * own_rows);
  l.own_wide = own_rows > 16;
  l.prefix_wide = prefix_rows > 16;
  size_t used = up256(sizeof(int32_t) * (size_t)(2 * a.B + 1));
  auto plan = [&](Plan& p, bool wide, bool prefix, bool own) {
    const int rows = prefix ? prefix_rows : own_rows;
    p.G = G;
    p.own_rows = own_rows;
    p.prefix_rows = prefix_rows;
    p.split_keys = wide && (!a.half || rows <= 128);
    p.rt = wide ? (p.split_keys ? 128 : 256) : a.half && rows > 8 ? 16 : 8;
    p.slot_rows = wide ? 256 : p.rt;
    p.subs = p.split_keys ? 2 : 1;
    p.unit = wide ? kTile : narrow_keys(a);
    p.own_nrt = own ? (own_rows + p.rt - 1) / p.rt : 0;
    p.prefix_nrt = prefix ? (prefix_rows + p.rt - 1) / p.rt : 0;
    const int tiles = prefix ? (int)((a.prefix_len + p.unit - 1) / p.unit) : 0;
    p.prefix_items = (int)a.own.heads * p.prefix_nrt;
    const int64_t own_items = a.B * a.own.heads * p.own_nrt;
    const int64_t most = (int64_t)p.prefix_items * tiles + own_items * ((a.own.max_seq + p.unit - 1) / p.unit);
    const int each = wide ? 1 : kWarps, full = kSms * (wide ? 1 : kNarrowCtas);  // workers of a CTA, CTAs
    p.grid = (int)(most < full * each ? (most + each - 1) / each : full);
    p.workers = p.grid * each;
    // A piece costs more than its keys (sums out, other queries in), so every item counts as kWideLead tiles or
    // kNarrowLead steps longer.  With 0, 3, 7 and 9 tiles 64 sequences behind 8192 positions take 55.5, 51.6, 49.3 and
    // 49.4 us, 24 x 4 tokens behind 4101 66.0, 48.5, 44.9 and 46.6, 128 sequences behind 32801 129.1, 125.2, 123.9 and
    // 123.2; with 0, 1, 2 and 4 steps 32 sequences of 4096 own positions 59.9, 58.3, 58.0 and 58.3, 64 behind 8192 52.7,
    // 49.4, 49.3 and 49.5.
    p.lead = wide ? kWideLead : kNarrowLead;
    p.prefix_units = tiles ? tiles + p.lead : 0;
    l.most = std::max(l.most, most + p.lead * (p.prefix_items + own_items));
    p.by_G = Div(G);
    p.by_rt = Div(p.rt);
    p.by_own_rows = Div(own_rows);
    p.by_own_nrt = Div(std::max(1, p.own_nrt));
    p.by_prefix_nrt = Div(std::max(1, p.prefix_nrt));
    p.by_prefix_units = Div(std::max(1, p.prefix_units));
    p.by_workers = Div(std::max(1, p.workers));
    const int64_t slot_rows = (p.prefix_items + own_items + p.workers) * p.slot_rows;
    p.part = reinterpret_cast<float*>(ws + used);
    used += up256(sizeof(float) * (size_t)(slot_rows * a.own.hd));
    p.ml = reinterpret_cast<float*>(ws + used);
    used += up256(sizeof(float) * (size_t)(slot_rows * 2));
  };
  if (l.own_wide) {
    plan(l.own, true, a.prefix_len > 0, true);
  } else {
    if (a.prefix_len) plan(l.prefix, l.prefix_wide, true, false);
    plan(l.own, false, false, true);
  }
  l.bytes = used;
  return l;
}

bool make_maps(Maps* m, const PrefixAttnArgs& a, int keys) {
  return make_map(&m->ok, a.own, a.own.k, keys) && make_map(&m->ov, a.own, a.own.v, keys) &&
         (!a.prefix_len || (make_map(&m->pk, a.prefix, a.prefix.k, keys) && make_map(&m->pv, a.prefix, a.prefix.v, keys)));
}

// `early`: launched when the grid before has started; it waits where it needs that one's results.
template <typename K, typename... Args>
cudaError_t launch(K kern, unsigned grid, int threads, int smem, bool early, cudaStream_t st, const Args&... args) {
  if (smem) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int F, int HD>
cudaError_t run_all(const PrefixAttnArgs& a, const Layout& l, const int32_t* given, int32_t* cum, cudaStream_t st) {
  Maps maps;
  auto wide = [&](const Plan& p) -> cudaError_t {
    if (!make_maps(&maps, a, kTile)) return cudaErrorInvalidValue;
    return launch(a.half ? wide_attn_kernel<F, HD, __half> : wide_attn_kernel<F, HD, float>, (unsigned)p.grid, Wide<F, HD>::kThreads,
                  Wide<F, HD>::kSmem, false, st, a, p, maps, given, cum);
  };
  auto narrow = [&](const Plan& p, bool early) -> cudaError_t {
    if (!make_maps(&maps, a, Narrow<F, HD>::kKeys)) return cudaErrorInvalidValue;
    const auto kern = !a.half      ? narrow_attn_kernel<F, HD, true, float>
                      : p.rt == 16 ? narrow_attn_kernel<F, HD, false, __half>
                                   : narrow_attn_kernel<F, HD, true, __half>;
    return launch(kern, (unsigned)p.grid, 32 * kWarps, Narrow<F, HD>::kSmem, early, st, a, p, maps, given, cum);
  };
  cudaError_t e = cudaSuccess;
  if (l.prefix.grid) e = l.prefix_wide ? wide(l.prefix) : narrow(l.prefix, false);
  if (e == cudaSuccess) e = l.own_wide ? wide(l.own) : narrow(l.own, l.prefix.grid > 0);
  if (e != cudaSuccess) return e;
  // four warps a row up to what the GPU holds at once (2048 rows 49.3 against 50.8 us with one; 4096 rows 129 against 124)
  const int64_t rows = a.B * a.T * a.H;
  const bool few = rows <= 16 * kSms;
  const auto kern = a.half ? (few ? join_kernel<HD, __half, 4> : join_kernel<HD, __half, 1>)
                           : (few ? join_kernel<HD, float, 4> : join_kernel<HD, float, 1>);
  const int32_t* sums = cum;
  return launch(kern, (unsigned)(few ? rows : (rows + 3) / 4), 128, 0, true, st, a, l.of_prefix(), l.own, sums);
}

template <int F>
cudaError_t run_dim(const PrefixAttnArgs& a, const Layout& l, const int32_t* given, int32_t* cum, cudaStream_t st) {
  return a.own.hd == 128 ? run_all<F, 128>(a, l, given, cum, st) : run_all<F, 64>(a, l, given, cum, st);
}

}  // namespace
}  // namespace attn

size_t prefix_attn_ws(const PrefixAttnArgs& a) { return attn::lay_out(a, nullptr).bytes; }

cudaError_t launch_prefix_attn(PrefixAttnArgs a, void* ws, int* launches, cudaStream_t st) {
  using namespace attn;
  const int64_t per16 = a.half ? 8 : 4;
  a.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.qs.batch % per16 == 0 && a.qs.token % per16 == 0 &&
            a.qs.head % per16 == 0;
  const Layout l = lay_out(a, static_cast<char*>(ws));
  if (l.most >= (int64_t(1) << 30)) return cudaErrorInvalidValue;  // (a cache of 2^35 positions)
  int32_t* cum = static_cast<int32_t*>(ws);
  const int32_t* given = nullptr;
  *launches = 2 + (l.prefix.grid > 0);
  if (a.B > kMaxScan) {
    sequences_kernel<<<1, 1024, 0, st>>>(a, l.own.unit, l.own.lead, cum);
    given = cum;
    ++*launches;
  }
  if (a.own.fmt == kKvI8) return run_dim<kKvI8>(a, l, given, cum, st);
  if (a.own.fmt == kKvE4M3) return run_dim<kKvE4M3>(a, l, given, cum, st);
  return run_dim<kKvF16>(a, l, given, cum, st);
}

}  // namespace uaii_b200
