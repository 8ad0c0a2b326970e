// serve_kernels.hpp -- launch wrappers of the serving operators around the decoder: the KV cache in
// f16 or 8 bits (kv_cache.cu), attention over a shared prefix and each sequence's own positions
// (prefix_attn.cu) and token sampling (sample.cu).  Plain pointers, sizes and a stream; each returns a
// cudaError_t.  Arguments are checked by the callers (serve.cpp, decoder.cpp).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace uaii_b200 {

// Formats of a KV cache: f16 values, or one byte per value and one f32 scale per row of head_dim values
// (value = (byte - 128) * scale, or e4m3(byte) * scale).  The values of the C ABI.
enum KvFormat { kKvF16 = 1, kKvI8 = 32, kKvE4M3 = 33 };

// (sequence, kv head) planes of a cache: one dimension of a grid.
constexpr int64_t kKvMaxPlanes = 65535;

// Codes in the backend's device error word for arguments that only the device can see.
constexpr int kErrKvPosition = 32;  // kv_append: a position outside the cache
constexpr int kErrKvLength = 33;    // attention: a length outside the cache
constexpr int kErrKvCopy = 34;      // attention: a copy of cached positions did not complete in time

// k, v [batch, n_kv_heads, max_seq, head_dim] (f16 or bytes), scales [batch, n_kv_heads, max_seq] or null.
struct KvCache {
  int fmt = 0;
  int hd = 0;
  int64_t batch = 0, heads = 0, max_seq = 0;
  void* k = nullptr;
  void* v = nullptr;
  float* k_scale = nullptr;
  float* v_scale = nullptr;
};

// Element strides of a [batch, token, head, head_dim] view whose last dimension is contiguous.
struct RowView {
  int64_t batch = 0, token = 0, head = 0;
};

// Tokens t < n_new[b] (all T when null) of k and v (f16 when half, else f32) into positions pos[b] + t.
cudaError_t launch_kv_append(const KvCache& c, const void* k, const void* v, bool half, int64_t T, const RowView& s,
                             const int32_t* pos, const int32_t* n_new, int* err, cudaStream_t st);
// Positions [pos0, pos0 + n) of every (sequence, head) as f32 or f16 [batch, heads, n, head_dim].
cudaError_t launch_kv_read(const KvCache& c, int64_t pos0, int64_t n, void* k_out, void* v_out, bool half,
                           cudaStream_t st);

// q and out f16 (half) or f32; out [B, T, H, hd] dense.  Token t of sequence b sees prefix positions
// [0, prefix_len) and own positions [0, own_len[b] - T + t].
struct PrefixAttnArgs {
  KvCache prefix, own;  // prefix.k null: none
  int64_t prefix_len = 0;
  const int32_t* own_len = nullptr;
  const void* q = nullptr;
  bool half = false;
  bool q_vec = false;  // every row of q starts on a 16-byte boundary (set by launch_prefix_attn)
  int64_t B = 0, T = 0, H = 0;
  RowView qs;
  float scale = 0.f;
  void* out = nullptr;
  int* err = nullptr;
};
size_t prefix_attn_ws(const PrefixAttnArgs& a);
cudaError_t launch_prefix_attn(PrefixAttnArgs a, void* ws, int* launches, cudaStream_t st);

// A row's weights lie in the shared memory of eight SMs.
constexpr int64_t kSampleMaxVocab = 8 * 50000;
// One token per row of logits [B, V] (f16 when half, else f32; rows ld elements apart); probs and kept may be null.
cudaError_t launch_sample(const void* logits, bool half, int64_t B, int64_t V, int64_t ld, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tokens,
                          float* probs, int32_t* kept, cudaStream_t st);

}  // namespace uaii_b200
