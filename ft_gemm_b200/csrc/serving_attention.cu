// Attention of each sequence's queries over its keys, packed or in the pages of a cache.
//
// Simple form: one warp per query row and head; 32 keys at a time, one per lane for the scores, then every lane
// accumulates its share of the head dimension.  All arithmetic in FP32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving_kernels.h"

namespace ftg {

namespace {

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_float(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

constexpr int kWarps = 8;

template <typename T, int kDim>
__global__ void __launch_bounds__(kWarps * 32) serve_attention_simple_kernel(const ServeAttentionParams p) {
  __shared__ float query[kWarps][kDim];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int head = blockIdx.y;
  const int token = blockIdx.x * kWarps + warp;
  const int total = min(p.q_offsets[p.batch], p.query_tokens);
  if (token >= total) return;
  int b = 0, hi = p.batch;  // the sequence of this token: the last whose offset is not behind it
  while (hi - b > 1) {
    const int mid = (b + hi) / 2;
    if (p.q_offsets[mid] <= token) b = mid; else hi = mid;
  }
  const int q_begin = p.q_offsets[b], queries = p.q_offsets[b + 1] - q_begin, row = token - q_begin;
  const bool paged = p.page_table != nullptr;
  int k_begin = 0, keys = 0;
  if (paged) {
    keys = min(p.lengths[b], p.table_pages * p.page_size);
  } else {
    k_begin = p.k_offsets[b];
    keys = min(p.k_offsets[b + 1], p.key_tokens) - k_begin;
  }
  const int prefix = (paged ? p.lengths[b] : keys) - queries;  // keys in front of the first query's own
  const T* q = reinterpret_cast<const T*>(p.q) + token * p.q_token_stride + head * p.q_head_stride;
  for (int d = lane; d < kDim; d += 32) query[warp][d] = to_float(q[d]) * p.scale_log2;
  __syncwarp();
  const int kv_head = head / p.group;
  const uint32_t* mask = p.mask == nullptr ? nullptr : p.mask + static_cast<long long>(token) * p.mask_stride;
  float top = -INFINITY, sum = 0.0f, o[kDim / 32] = {};
  for (int key0 = 0; key0 < keys; key0 += 32) {
    const int key = key0 + lane;
    bool visible = key < keys;
    if (visible && key >= prefix) {
      const int node = key - prefix;
      if (mask != nullptr) {
        visible = node < p.mask_words * 32 && ((mask[node / 32] >> (node % 32)) & 1) != 0;
      } else if (p.causal) {
        visible = node <= row;
      }
    }
    long long at = 0, v_at = 0;
    if (visible) {
      if (paged) {
        const int page = p.page_table[static_cast<long long>(b) * p.table_stride + key / p.page_size];
        if (page < 0 || page >= p.pages) {
          at = v_at = -1;
        } else {
          at = v_at = page * p.page_stride + (key % p.page_size) * p.kv_token_stride + kv_head * p.kv_head_stride;
        }
      } else {
        at = (k_begin + key) * p.kv_token_stride + kv_head * p.kv_head_stride;
        v_at = (k_begin + key) * p.v_token_stride + kv_head * p.v_head_stride;
      }
    }
    float score = -INFINITY;
    if (visible) {
      score = 0.0f;
      if (at >= 0) {
        for (int d = 0; d < kDim; ++d) score = fmaf(query[warp][d], to_float(reinterpret_cast<const T*>(p.k)[at + d]), score);
      }
    }
    float best = score;
    for (int off = 16; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, off));
    const float next = fmaxf(top, best);
    const float reference = next == -INFINITY ? 0.0f : next;  // nothing seen so far; a NaN score stays one
    const float shrink = exp2f(top - reference);
    const float e = visible ? exp2f(score - reference) : 0.0f;
    float s = e;
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    sum = sum * shrink + s;
    top = next;
    for (int i = 0; i < kDim / 32; ++i) o[i] *= shrink;
    for (int j = 0; j < 32; ++j) {
      const float w = __shfl_sync(0xffffffffu, e, j);
      const long long from = __shfl_sync(0xffffffffu, v_at, j);
      if (__shfl_sync(0xffffffffu, visible ? 1 : 0, j) == 0 || from < 0) continue;
      for (int i = 0; i < kDim / 32; ++i) o[i] = fmaf(w, to_float(reinterpret_cast<const T*>(p.v)[from + i * 32 + lane]), o[i]);
    }
  }
  T* out = reinterpret_cast<T*>(p.out) + token * p.out_token_stride + head * p.out_head_stride;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int i = 0; i < kDim / 32; ++i) from_float(out[i * 32 + lane], o[i] * inv);
  if (p.lse != nullptr && lane == 0) p.lse[static_cast<long long>(token) * p.heads + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace

cudaError_t launch_serve_attention(const ServeAttentionParams& p, int dtype, cudaStream_t stream) {
  if (p.query_tokens <= 0 || p.batch <= 0) return cudaSuccess;
  const dim3 grid((p.query_tokens + kWarps - 1) / kWarps, p.heads);
  if (dtype == FT_SRC_BF16) {
    if (p.head_dim == 128) serve_attention_simple_kernel<__nv_bfloat16, 128><<<grid, kWarps * 32, 0, stream>>>(p);
    else serve_attention_simple_kernel<__nv_bfloat16, 64><<<grid, kWarps * 32, 0, stream>>>(p);
  } else {
    if (p.head_dim == 128) serve_attention_simple_kernel<__half, 128><<<grid, kWarps * 32, 0, stream>>>(p);
    else serve_attention_simple_kernel<__half, 64><<<grid, kWarps * 32, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace ftg
