/*
 * ft_serving.h -- C-ABI of the operators a decoder needs around its attention when
 * it is served: rotary positions, a paged key/value cache, attention over packed
 * prompts of different lengths, and attention of drafted tokens (a single new token
 * among them) over the cache.  The reference project has none of them; they stand
 * beside the protected attention of ft_attention.h and share its error codes and
 * ft_gemm_last_error().
 *
 * Common rules.  Element types are FT_SRC_BF16 and FT_SRC_F16 (ft_gemm.h); sums and
 * softmax statistics are held in 32 bits, angles formed in 64, and every result is
 * rounded once.  The attention also rounds each probability once, to the element type,
 * as an operand of its second product (the denominator adds them up before that).
 * All pointers inside the structures are device pointers unless a field says "host".
 * Calls are asynchronous on `stream`, allocate nothing, keep nothing between calls and
 * may be captured into a graph; two calls may run at the same time on different streams
 * when they write different memory (workspaces included).  They run on the calling
 * thread's current device.
 */
#ifndef FT_SERVING_H
#define FT_SERVING_H

#include <stddef.h>
#include <stdint.h>

#include "ft_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows [token][head][head_dim], head_dim contiguous.  `data` and both strides (in
 * elements) must be multiples of 16 bytes, so slices of a fused QKV projection fit. */
typedef struct {
  void* data;
  long long token_stride;
  long long head_stride;
  int heads;
} ft_rows;

/* ---- rotary positions ----------------------------------------------------------
 * Pair i of a head at position p turns by p * f_i:
 *   (a, b) -> magnitude * (a cos - b sin, a sin + b cos)
 * with the pairs (i, i + rotary_dim/2), or (2i, 2i + 1) when interleaved; the
 * elements from rotary_dim on are copied.  f_i = base^(-2 i / rotary_dim), scaled for
 * long contexts by one of FT_ROTARY_*.  Frequencies are doubles, an angle is one product and
 * one reduction in 64 bits: off by 2^-52 of its turns (p * f_i / 2pi), which after 2^24 of them
 * (positions of 100 million) is still less than the rounding of its sine in 32 bits. */
#define FT_ROTARY_PLAIN 0
#define FT_ROTARY_LINEAR 1   /* f_i / factor */
#define FT_ROTARY_BASE 2     /* base * factor^(rotary_dim / (rotary_dim - 2)) */
#define FT_ROTARY_BY_PARTS 3 /* with turns t = original_length * f_i / 2pi and g = clamp((t - low) / (high - low), 0, 1): f_i * (g + (1 - g) / factor) */

typedef struct {
  int head_dim;   /* a multiple of 16, at most 256 */
  int rotary_dim; /* a multiple of 16, at most head_dim */
  int interleaved;
  int scaling;
  double base;            /* default 10000 */
  double factor;          /* default 1 */
  double original_length; /* FT_ROTARY_BY_PARTS only */
  double low, high;       /* default 1, 4: turns within the original length below which f is divided, above which it is kept */
  double magnitude;       /* default 1 */
} ft_rotary_options;

typedef struct ft_rotary_handle ft_rotary_handle;

void ft_rotary_options_default(ft_rotary_options* options, int head_dim);

/* The rotary_dim/2 frequencies in radians per position, into host memory. */
int ft_rotary_frequencies(const ft_rotary_options* options, double* host_out);

/* The handle holds the frequencies on the current device and is not written by runs.  Captured graphs
 * read it too: it is destroyed after them. */
int ft_rotary_prepare(ft_rotary_handle** handle, const ft_rotary_options* options, void* stream);
int ft_rotary_destroy(ft_rotary_handle* handle);

/* Rotates q and k (k may be NULL) at positions[token].  An output may be its input
 * (the same data and strides); other overlaps are not allowed, and the rows of an output must not share
 * memory (inputs may: a broadcast head).  inverse != 0 turns
 * back (times magnitude once more), which is also the gradient: pass the output gradients
 * as q and k.  Rows at or behind `tokens` are neither read nor written.  At most 2^30
 * tokens and 2^20 heads. */
int ft_rotary_run(const ft_rotary_handle* handle, const ft_rows* q, const ft_rows* q_out, const ft_rows* k, const ft_rows* k_out,
                  const long long* positions, int tokens, int dtype, int inverse, void* stream);

/* ---- paged key/value cache -------------------------------------------------------
 * K and V of `layers` layers: element (layer, page, token in page, head, d) lies at
 * layer * layer_stride + page * page_stride + token * token_stride + head * head_stride + d.
 * Strides are in elements, multiples of 16 bytes, the same for K and V; no two pages of
 * any layers share memory (layers may lie between pages); a page of a layer is dense in either order: (token_stride, head_stride) = (kv_heads * head_dim,
 * head_dim) or (head_dim, page_size * head_dim).  For the attention page_stride is a
 * multiple of 8 * token_stride, as it is for dense pages and for pages of K and V in turn.
 * K and V must not share memory, except that one slab may be read as both (k == v) by the
 * attention; appending to it and accepting in it are refused. */
typedef struct {
  void* k;
  void* v;
  long long layer_stride, page_stride, token_stride, head_stride;
  int layers, pages;
  int page_size; /* a power of two from 8 to 256 */
  int kv_heads; /* at most 8192 */
  int head_dim; /* 64 or 128 */
  int dtype;
} ft_kv_cache;

/* Writes k and v of `tokens` tokens to slots[token] = page * page_size + token in page of
 * one layer.  A token whose slot is negative or behind the last page is not written
 * (padding of a batch); the slots of one call must differ.  With `rotary`, k is rotated at
 * positions[token] on the way, and q (may be NULL) is rotated into q_out in the same pass
 * (q_out may be q; its rows must not share memory). */
int ft_kv_cache_append(const ft_kv_cache* cache, int layer, const ft_rows* k, const ft_rows* v, const long long* slots, int tokens,
                       const ft_rotary_handle* rotary, const long long* positions, const ft_rows* q, const ft_rows* q_out, void* stream);

/* Copies page sources[i] to page targets[i] in every layer.  No target may be a source or
 * another target of the same call; pairs that name a page outside the cache are ignored.  More
 * than 2^31 - 1 pieces of 16 KiB in all (count times those of a page) are refused. */
int ft_kv_cache_copy_pages(const ft_kv_cache* cache, const int* sources, const int* targets, int count, void* stream);

/* Keeps the accepted ones of each sequence's drafted tokens: sequence b holds lengths[b]
 * tokens, the last n_b = drafted_offsets[b+1] - drafted_offsets[b] of them drafted.  Drafted
 * token accepted[accepted_offsets[b] + i] (ascending in i) moves to place lengths[b] - n_b + i in
 * every layer, and new_lengths[b] (not the same array as lengths) becomes lengths[b] - n_b +
 * the number accepted.  page_table[b * table_stride + j] is the page of tokens
 * [j, j + 1) * page_size of sequence b, j < table_pages.  Offsets ascend, and the pages of the
 * drafted tokens belong to one sequence only.  Moves that name a place outside the drafted tokens
 * or a page outside the cache are left out. */
int ft_kv_cache_accept(const ft_kv_cache* cache, const int* page_table, int table_pages, int table_stride, const int* lengths,
                       const int* drafted_offsets, const int* accepted, const int* accepted_offsets, int batch, int* new_lengths, void* stream);

/* ---- page pool (host) ------------------------------------------------------------
 * Which sequence holds which page.  A forked sequence shares its pages with its parent
 * until one of them writes: _extend then gives the writer a copy of the last, partly
 * filled page.  (Places that both held when they were forked stay shared: they are written before
 * the fork.)  Calls that move contents return the pairs to hand to
 * ft_kv_cache_copy_pages before the next append, and before _free or _truncate give a page
 * back that one of the pairs names.  One thread at a time. */
typedef struct ft_page_pool ft_page_pool;

int ft_page_pool_create(ft_page_pool** pool, int pages, int page_size);
int ft_page_pool_destroy(ft_page_pool* pool);
int ft_page_pool_free_pages(const ft_page_pool* pool); /* or a negative error code */
int ft_page_pool_new_sequence(ft_page_pool* pool, int* sequence);
int ft_page_pool_fork(ft_page_pool* pool, int sequence, int* child);
int ft_page_pool_free(ft_page_pool* pool, int sequence);
/* Appends `tokens` places; FT_ERR_INVALID, with nothing changed, when the pages do not suffice.
 * *source is -1, or the page to copy to *target. */
int ft_page_pool_extend(ft_page_pool* pool, int sequence, int tokens, int* source, int* target);
int ft_page_pool_truncate(ft_page_pool* pool, int sequence, int length);
int ft_page_pool_length(const ft_page_pool* pool, int sequence); /* or a negative error code */
/* The pages of a sequence, up to `capacity` of them, into host memory; returns their number or an error. */
int ft_page_pool_pages(const ft_page_pool* pool, int sequence, int* host_pages, int capacity);
/* Moves the used pages to the front of the cache: at most `capacity` pairs (sources, targets) in
 * host memory; *count is their number.  No target is a source. */
int ft_page_pool_compact(ft_page_pool* pool, int* host_sources, int* host_targets, int capacity, int* count);

/* ---- attention --------------------------------------------------------------------
 * out = softmax(scale * q k^T over the visible keys) v, per query head; query head h reads
 * key head h / (heads / kv_heads), at most 128 query heads per key head.  A row that sees no
 * key gives zeros (and lse -inf).  head_dim is 64 or 128.  lse (may be NULL) is
 * float [token][head], the natural logarithm of the softmax denominator.  Output rows behind the
 * last sequence are left as they are.  `out` and lse overlap no input.  Packed k and v have at most
 * 2^27 rows, and a page table holds at most 2^27 tokens.  A call has at most some 2^31 tiles of 128
 * rows by 128 keys: counted with table_pages for each sequence over the cache, and with all of q and k
 * for a single packed sequence, and refused beyond; several packed sequences are counted on the device,
 * each with its own keys, and where they pass it the call writes FT_ERR_INVALID to `status` and no output.
 *
 * Values are added up in 32 bits by the tensor core, which cuts products off towards zero: over N
 * keys by at most N 2^-27 of the sum, and never more than 2^-10.
 *
 * What lies behind a sequence's last key never reaches its output, whatever it is.  A key that some
 * rows of a sequence see and others do not has the probability zero in the others: K may hold
 * anything there, but a NaN or an infinity in V can reach rows that do not see it (zero times V).
 *
 * `workspace` holds ft_attention_workspace() bytes, 16-byte aligned, contents arbitrary; calls that
 * can run at the same time need one each.  `status` is an int the caller sets to zero once; a
 * device-side wait that gives up writes FT_ERR_TIMEOUT there (the output is then not valid), too many
 * packed tiles FT_ERR_INVALID, and nothing ever clears it. */
size_t ft_attention_workspace(void);

/* Packed prompts: sequence b has the queries q_offsets[b] .. q_offsets[b+1] and the keys
 * k_offsets[b] .. k_offsets[b+1] (k_offsets NULL: the same).  causal: the last query sees every
 * key of its sequence, the query before it all but the last key, and so on.  Offsets ascend from 0. */
typedef struct {
  ft_rows q, k, v, out;
  float* lse;
  const int* q_offsets;
  const int* k_offsets;
  int batch;
  int query_tokens, key_tokens; /* rows that q / out and k / v hold */
  int head_dim, dtype, causal;
  float scale; /* 0: 1 / sqrt(head_dim) */
} ft_prompt_attention_args;

int ft_prompt_attention_run(const ft_prompt_attention_args* args, void* workspace, size_t workspace_bytes, int* status, void* stream);

/* Drafted tokens over the cache: sequence b holds lengths[b] tokens in the pages of row b of
 * page_table ([batch][table_stride], table_pages of each row valid); its last n_b = q_offsets[b+1] -
 * q_offsets[b] are the drafted ones, whose K and V are already in the cache and whose queries are q.
 * Every query sees all tokens before the drafted ones, and drafted token j if bit j of its mask row
 * (32-bit words, mask_stride words from row to row, mask_words valid) is set; mask NULL: j up to
 * itself, a chain (n_b = 1: plain decoding; larger: a piece of a prompt over its cached start).
 * What the cache holds behind lengths[b] is not looked at.  A page number outside the cache reads as
 * zeros. */
typedef struct {
  ft_rows q, out;
  float* lse;
  const int* q_offsets;
  const int* page_table;
  const int* lengths;
  const uint32_t* mask;
  int mask_words, mask_stride;
  int batch, query_tokens;
  int table_pages, table_stride;
  int layer;
  float scale; /* 0: 1 / sqrt(head_dim) */
} ft_tree_attention_args;

int ft_tree_attention_run(const ft_kv_cache* cache, const ft_tree_attention_args* args, void* workspace, size_t workspace_bytes, int* status,
                          void* stream);

/* Mask rows of a tree from its parents (host memory): parents[i] < i, or negative for a root; bit j of
 * row i is set when j is i or an ancestor of i.  `words` must hold `nodes` bits. */
int ft_tree_mask(const int* host_parents, int nodes, uint32_t* host_mask, int words);

#ifdef __cplusplus
}
#endif
#endif
