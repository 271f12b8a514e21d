// Internal interface between the serving C-ABI (api_serving.cu) and its kernels.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/ft_serving.h"

namespace ftg {

struct Rows {  // ft_rows with 16-bit elements
  uint16_t* data;
  long long token_stride, head_stride;
};

// One pass over the rows of a token: rotates q and k (or copies them where rotary_dim ends), writes k and v to pages.
struct RotaryParams {
  Rows q, q_out, k, k_out, v;
  int q_heads, k_heads, v_heads;  // v_heads: k_heads when K and V go to the cache, else 0
  const double* turns;            // frequencies in turns per position, rotary_dim / 2 of them
  const long long* positions;
  const long long* slots;  // with the cache: where k and v go
  uint16_t *k_cache, *v_cache;
  long long page_stride, cache_token_stride, cache_head_stride;
  long long slot_count;
  int page_shift;  // page_size = 1 << page_shift
  int tokens, head_dim, rotary_dim;
  int interleaved, inverse;
  float magnitude;
};
cudaError_t launch_rotary(const RotaryParams& params, int dtype, cudaStream_t stream);

struct CopyPagesParams {
  uint16_t *k, *v;
  long long layer_stride, page_stride;
  int layers, pages, page_elements, count;
  const int *sources, *targets;
};
int copy_pages_most(int page_elements);  // pairs of one call
cudaError_t launch_copy_pages(const CopyPagesParams& params, cudaStream_t stream);

struct AcceptParams {
  uint16_t *k, *v;
  long long layer_stride, page_stride, token_stride, head_stride;
  int layers, pages, page_size, kv_heads, head_dim;
  const int *page_table, *lengths, *drafted_offsets, *accepted, *accepted_offsets;
  int table_pages, table_stride, batch;
  int* new_lengths;
};
cudaError_t launch_accept(const AcceptParams& params, cudaStream_t stream);

// Attention of the queries of each sequence over its keys: packed prompts (page_table == nullptr) or the paged cache.
struct ServeAttentionParams {
  uint16_t* out;
  float* lse;
  long long out_token_stride, out_head_stride;
  const int* q_offsets;
  const int* k_offsets;   // packed prompts
  const int* page_table;  // paged cache
  const int* lengths;
  const uint32_t* mask;
  int mask_words, mask_stride;
  int batch, query_tokens, key_tokens;
  int heads, kv_heads, group, head_dim, causal;
  int tokens_per_tile;  // 128 / group: tokens whose heads fill a tile of 128 rows
  int page_size, pages, table_pages, table_stride;
  int page_groups;   // groups of 8 tokens from page to page
  int count_units;   // the host could not tell that the units of work stay inside 31 bits
  float scale_log2;  // log2(e) * scale
  void* workspace;
  int* status;
};
size_t serve_attention_workspace(int sm_count);
// q: [token][key head][head in group][d], boxes of 128 / group tokens; k, v: [token][key head][d] in boxes of 128 tokens, or
// [key head][8 tokens][64 elements][token in 8][element] in boxes of up to 128 tokens of a page, the pages page_groups groups of 8 apart.  split_keys: one row tile per CTA, the two warpgroups
// take turns on its key tiles.
cudaError_t launch_serve_attention(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ServeAttentionParams& params, int dtype,
                                   bool split_keys, int sm_count, cudaStream_t stream);

}  // namespace ftg
