// serve.cpp -- the serving operators around the decoder: argument checks, and the extern "C" shim of the KV cache
// (f16 or 8 bits), attention over a shared prefix, and sampling (include/uaii_moe.h).  Every pointer is device
// memory; work is queued on the backend's stream and a call returns without waiting.  What only the device can see
// (a position or a length outside the cache) is skipped there and reported by the next synchronization.
#include <cmath>
#include <exception>
#include <string>

#include "../../include/uaii_moe.h"
#include "backend.hpp"
#include "serve_kernels.hpp"

namespace uaii_b200 {

namespace {

Error invalid(const std::string& what) { return Error::make(ErrorCode::InvalidArgument, what); }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxCount = int64_t(1) << 31;  // grids and table entries are 32 bits

Error check_dtype(const char* op, int dtype, bool* half) {
  if (dtype != UAII_MOE_DTYPE_F32 && dtype != UAII_MOE_DTYPE_F16)
    return Error::make(ErrorCode::NotImplemented, std::string(op) + ": dtype must be f32 or f16");
  *half = dtype == UAII_MOE_DTYPE_F16;
  return Error::success();
}

}  // namespace

Error kv_cache_from_c(const char* op, const uaii_moe_kv_cache* s, KvCache* out) {
  const std::string o(op);
  if (!s) return invalid(o + ": null cache");
  if (s->fmt != kKvF16 && s->fmt != kKvI8 && s->fmt != kKvE4M3)
    return Error::make(ErrorCode::NotImplemented, o + ": cache format must be F16, KV_I8 or KV_E4M3");
  if (s->head_dim != 64 && s->head_dim != 128)
    return Error::make(ErrorCode::NotImplemented, o + ": head_dim must be 64 or 128");
  if (s->batch <= 0 || s->n_kv_heads <= 0 || s->max_seq <= 0 || s->batch >= kMaxCount || s->n_kv_heads >= kMaxCount ||
      s->max_seq >= kMaxCount || s->batch > kKvMaxPlanes || s->batch * s->n_kv_heads > kKvMaxPlanes)
    return invalid(o + ": cache sizes out of range");
  if (!is_device_ptr(s->k) || !is_device_ptr(s->v)) return invalid(o + ": the cache must be device memory");
  if (!aligned(s->k, 16) || !aligned(s->v, 16)) return invalid(o + ": the cache must start on a 16-byte boundary");
  if (s->fmt != kKvF16) {
    if (!is_device_ptr(s->k_scale) || !is_device_ptr(s->v_scale))
      return invalid(o + ": an 8-bit cache needs its row scales in device memory");
    if (!aligned(s->k_scale, 4) || !aligned(s->v_scale, 4)) return invalid(o + ": misaligned row scales");
  }
  out->fmt = s->fmt;
  out->hd = s->head_dim;
  out->batch = s->batch;
  out->heads = s->n_kv_heads;
  out->max_seq = s->max_seq;
  out->k = s->k;
  out->v = s->v;
  out->k_scale = s->fmt == kKvF16 ? nullptr : s->k_scale;
  out->v_scale = s->fmt == kKvF16 ? nullptr : s->v_scale;
  return Error::success();
}

Error check_sample_arrays(const char* op, const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                          const float* u, const int32_t* tokens, const float* probs, const int32_t* kept) {
  const void* needed[] = {temperature, top_k, top_p, min_p, u, tokens};
  const void* optional[] = {probs, kept};
  for (const void* p : needed) {
    if (!is_device_ptr(p)) return invalid(std::string(op) + ": arguments must be device memory");
    if (!aligned(p, 4)) return invalid(std::string(op) + ": misaligned argument");
  }
  for (const void* p : optional) {
    if (p && !is_device_ptr(p)) return invalid(std::string(op) + ": arguments must be device memory");
    if (!aligned(p, 4)) return invalid(std::string(op) + ": misaligned argument");
  }
  return Error::success();
}

Error MoeCudaBackend::kv_append(const KvCache& c, const void* k, const void* v, bool half, int64_t T, const RowView& s,
                                const int32_t* pos, const int32_t* n_new) {
  std::lock_guard<std::mutex> lk(mu_);
  if (T < 0 || T > c.max_seq) return invalid("kv_append: token count out of range");
  if (T == 0) return Error::success();
  if (!is_device_ptr(k) || !is_device_ptr(v) || !is_device_ptr(pos) || (n_new && !is_device_ptr(n_new)))
    return invalid("kv_append: arguments must be device memory");
  const size_t esz = half ? 2 : 4;
  if (!aligned(k, esz) || !aligned(v, esz) || !aligned(pos, 4) || !aligned(n_new, 4))
    return invalid("kv_append: misaligned argument");
  if (c.batch * c.heads * T >= kMaxCount) return invalid("kv_append: too many rows for one call");
  UAII_CUDA(cudaSetDevice(device_), "SetDevice");
  UAII_CUDA(launch_kv_append(c, k, v, half, T, s, pos, n_new, dev_err_, stream_), "kv_append");
  count_launches(1);
  return Error::success();
}

Error MoeCudaBackend::kv_read(const KvCache& c, int64_t pos0, int64_t n, void* k_out, void* v_out, bool half) {
  std::lock_guard<std::mutex> lk(mu_);
  if (pos0 < 0 || n < 0 || pos0 > c.max_seq || n > c.max_seq - pos0) return invalid("kv_read: positions outside the cache");
  if (n == 0) return Error::success();
  if (!is_device_ptr(k_out) || !is_device_ptr(v_out)) return invalid("kv_read: outputs must be device memory");
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return invalid("kv_read: outputs must start on a 16-byte boundary");
  UAII_CUDA(cudaSetDevice(device_), "SetDevice");
  UAII_CUDA(launch_kv_read(c, pos0, n, k_out, v_out, half, stream_), "kv_read");
  count_launches(1);
  return Error::success();
}

Error MoeCudaBackend::prefix_attention(PrefixAttnArgs a) {
  std::lock_guard<std::mutex> lk(mu_);
  const char* op = "prefix_attention: ";
  if (a.T < 0 || a.H <= 0 || a.H % a.own.heads != 0)
    return invalid(std::string(op) + "n_tokens >= 0 and n_heads a multiple of the cache's n_kv_heads");
  a.B = a.own.batch;
  if (a.prefix_len < 0) return invalid(std::string(op) + "negative prefix length");
  if (a.prefix_len == 0) {
    a.prefix = KvCache{};
  } else {
    if (!a.prefix.k) return invalid(std::string(op) + "prefix_len without a prefix cache");
    if (a.prefix.fmt != a.own.fmt || a.prefix.hd != a.own.hd || a.prefix.heads != a.own.heads)
      return invalid(std::string(op) + "the prefix and own caches must share format, head_dim and n_kv_heads");
    if (a.prefix.batch != 1) return invalid(std::string(op) + "the prefix cache holds one sequence");
    if (a.prefix_len > a.prefix.max_seq) return invalid(std::string(op) + "prefix_len exceeds the prefix cache");
  }
  if (a.scale == 0.f) a.scale = 1.0f / std::sqrt((float)a.own.hd);
  if (!std::isfinite(a.scale)) return invalid(std::string(op) + "scale must be finite");
  if (a.T == 0) return Error::success();
  if (a.H >= kMaxCount || a.T >= kMaxCount || a.T * a.H >= kMaxCount || a.B * a.T * a.H >= kMaxCount)
    return invalid(std::string(op) + "too many query rows for one call");
  if (!is_device_ptr(a.q) || !is_device_ptr(a.own_len) || !is_device_ptr(a.out))
    return invalid(std::string(op) + "arguments must be device memory");
  const size_t esz = a.half ? 2 : 4;
  if (!aligned(a.q, esz) || !aligned(a.own_len, 4) || !aligned(a.out, 16))
    return invalid(std::string(op) + "misaligned argument (out starts on a 16-byte boundary)");
  UAII_CUDA(cudaSetDevice(device_), "SetDevice");
  a.err = dev_err_;
  const size_t ws = prefix_attn_ws(a);
  UAII_TRY(reserve(ws));
  int launches = 0;
  UAII_CUDA(launch_prefix_attn(a, ws ? carve(ws) : nullptr, &launches, stream_), "prefix_attention");
  count_launches((uint64_t)launches);
  return Error::success();
}

Error MoeCudaBackend::sample(const void* logits, bool half, int64_t B, int64_t V, int64_t ld, const float* temperature,
                             const int32_t* top_k, const float* top_p, const float* min_p, const float* u,
                             int32_t* tokens, float* probs, int32_t* kept) {
  std::lock_guard<std::mutex> lk(mu_);
  if (B < 0 || V <= 0 || V >= kMaxCount || B >= kMaxCount) return invalid("sample: batch >= 0 and 0 < vocab < 2^31");
  if (V > kSampleMaxVocab)
    return Error::make(ErrorCode::NotImplemented, "sample: vocab above " + std::to_string(kSampleMaxVocab));
  if (ld < V) return invalid("sample: rows overlap (ld < vocab)");
  if (B == 0) return Error::success();
  if (!is_device_ptr(logits)) return invalid("sample: arguments must be device memory");
  UAII_TRY(check_sample_arrays("sample", temperature, top_k, top_p, min_p, u, tokens, probs, kept));
  if (!aligned(logits, half ? 2 : 4)) return invalid("sample: misaligned logits");
  UAII_CUDA(cudaSetDevice(device_), "SetDevice");
  UAII_CUDA(launch_sample(logits, half, B, V, ld, temperature, top_k, top_p, min_p, u, tokens, probs, kept, stream_),
            "sample");
  count_launches(1);
  return Error::success();
}

}  // namespace uaii_b200

using namespace uaii_b200;

namespace {

// No C++ exception (a failed allocation of a message, a system error of a lock) leaves a C entry.
template <typename F>
int guarded(uaii_moe_backend* b, F&& f) {
  try {
    if (!b) return report_status(Error::make(ErrorCode::InvalidArgument, "null backend"));
    return report_status(f());
  } catch (const std::exception& e) {
    try {
      return report_status(Error::make(ErrorCode::Internal, e.what()));
    } catch (...) {
      return UAII_MOE_INTERNAL;
    }
  }
}

}  // namespace

extern "C" {

int uaii_moe_kv_append(uaii_moe_backend* b, const uaii_moe_kv_cache* cache, const void* k, const void* v, int dtype,
                       int64_t n_tokens, int64_t stride_batch, int64_t stride_token, int64_t stride_head,
                       const int32_t* pos, const int32_t* n_new) {
  return guarded(b, [&]() -> Error {
    KvCache c;
    bool half = false;
    UAII_TRY(kv_cache_from_c("kv_append", cache, &c));
    UAII_TRY(check_dtype("kv_append", dtype, &half));
    return b->impl.kv_append(c, k, v, half, n_tokens, RowView{stride_batch, stride_token, stride_head}, pos, n_new);
  });
}

int uaii_moe_kv_read(uaii_moe_backend* b, const uaii_moe_kv_cache* cache, int64_t pos0, int64_t n, void* k_out,
                     void* v_out, int dtype) {
  return guarded(b, [&]() -> Error {
    KvCache c;
    bool half = false;
    UAII_TRY(kv_cache_from_c("kv_read", cache, &c));
    UAII_TRY(check_dtype("kv_read", dtype, &half));
    return b->impl.kv_read(c, pos0, n, k_out, v_out, half);
  });
}

int uaii_moe_prefix_attention(uaii_moe_backend* b, const uaii_moe_kv_cache* prefix, int64_t prefix_len,
                              const uaii_moe_kv_cache* own, const int32_t* own_len, const void* q, int dtype,
                              int64_t n_heads, int64_t n_tokens, int64_t stride_batch, int64_t stride_token,
                              int64_t stride_head, float scale, void* out) {
  return guarded(b, [&]() -> Error {
    PrefixAttnArgs a;
    UAII_TRY(kv_cache_from_c("prefix_attention", own, &a.own));
    if (prefix) UAII_TRY(kv_cache_from_c("prefix_attention", prefix, &a.prefix));
    UAII_TRY(check_dtype("prefix_attention", dtype, &a.half));
    a.prefix_len = prefix_len;
    a.own_len = own_len;
    a.q = q;
    a.T = n_tokens;
    a.H = n_heads;
    a.qs = RowView{stride_batch, stride_token, stride_head};
    a.scale = scale;
    a.out = out;
    return b->impl.prefix_attention(a);
  });
}

int uaii_moe_sample(uaii_moe_backend* b, const void* logits, int dtype, int64_t batch, int64_t vocab, int64_t ld,
                    const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                    const float* u, int32_t* tokens, float* probs, int32_t* kept) {
  return guarded(b, [&]() -> Error {
    bool half = false;
    UAII_TRY(check_dtype("sample", dtype, &half));
    return b->impl.sample(logits, half, batch, vocab, ld, temperature, top_k, top_p, min_p, u, tokens, probs, kept);
  });
}

}  // extern "C"
