// C-ABI of the serving operators: see include/ft_serving.h.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <new>
#include <utility>
#include <vector>

#include "serving_kernels.h"

using namespace ftg;

namespace ftg {
int noalloc_fail(int code, const char* fmt, ...);  // sets the thread's last-error text (api.cu)
}

namespace {

#define SERVE_CUDA(call)                                                                                     \
  do {                                                                                                       \
    cudaError_t err_ = (call);                                                                               \
    if (err_ != cudaSuccess) return noalloc_fail(FT_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(err_)); \
  } while (0)

constexpr float kLog2E = 1.44269504088896340736f;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The rules every ft_rows has to meet; `heads` is what the operator expects there.
int check_rows(const ft_rows* r, const char* name, int heads) {
  if (r == nullptr || r->data == nullptr) return noalloc_fail(FT_ERR_INVALID, "null %s", name);
  if (r->heads != heads) return noalloc_fail(FT_ERR_INVALID, "%s has %d heads where %d are expected", name, r->heads, heads);
  if (!aligned16(r->data) || r->token_stride % 8 != 0 || r->head_stride % 8 != 0 || r->token_stride < 0 || r->head_stride < 0) {
    return noalloc_fail(FT_ERR_INVALID, "%s must be 16-byte aligned with strides that are multiples of 8 elements", name);
  }
  return FT_OK;
}

// The tensor-copy engine steps through rows that do not overlap: a broadcast head or token is refused.
int check_apart(const ft_rows* r, const char* name, int tokens, int head_dim) {
  if ((r->heads > 1 && r->head_stride < head_dim) || (tokens > 1 && r->token_stride < head_dim)) {
    return noalloc_fail(FT_ERR_INVALID, "the heads and tokens of %s must not share memory (strides %lld, %lld)", name, r->token_stride, r->head_stride);
  }
  return FT_OK;
}

// Do any two of the m * n blocks of `block` elements at i * a + j * b share memory?
bool blocks_meet(long long a, long long m, long long b, long long n, long long block) {
  if ((m > 1 && a < block) || (n > 1 && b < block)) return true;
  if (m <= 1 || n <= 1 || (b - block) / a >= m - 1 || (a - block) / b >= n - 1) return false;  // one dimension lies within a step of the other
  if (m > n) {
    std::swap(a, b);
    std::swap(m, n);
  }
  for (long long i = 1; i < m; ++i) {  // the two steps of b on either side of i * a
    const __int128 at = static_cast<__int128>(i) * a, j = at / b, past = at - j * b;
    if ((j >= 1 && j < n && past < block) || (j + 1 < n && b - past < block)) return true;
  }
  return false;
}

// Outputs are written by many threads at once: no two rows may share memory, and an output that is its input has its strides.
int check_output(const ft_rows* r, const char* name, int tokens, int head_dim, const ft_rows* input) {
  if (blocks_meet(r->head_stride, r->heads, r->token_stride, tokens, head_dim)) {
    return noalloc_fail(FT_ERR_INVALID, "the heads and tokens of %s must not share memory (strides %lld, %lld)", name, r->token_stride, r->head_stride);
  }
  if (input != nullptr && r->data == input->data &&
      ((r->heads > 1 && r->head_stride != input->head_stride) || (tokens > 1 && r->token_stride != input->token_stride))) {
    return noalloc_fail(FT_ERR_INVALID, "%s lies where its input does, with other strides", name);
  }
  return FT_OK;
}

int check_dtype(int dtype) {
  if (dtype != FT_SRC_BF16 && dtype != FT_SRC_F16) return noalloc_fail(FT_ERR_INVALID, "dtype must be FT_SRC_BF16 or FT_SRC_F16");
  return FT_OK;
}

Rows to_rows(const ft_rows* r) { return Rows{static_cast<uint16_t*>(r->data), r->token_stride, r->head_stride}; }

int check_cache(const ft_kv_cache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr) return noalloc_fail(FT_ERR_INVALID, "null cache, K or V");
  const int rc = check_dtype(c->dtype);
  if (rc != FT_OK) return rc;
  if (c->layers <= 0 || c->layers > 32767 || c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 8192 || (c->head_dim != 64 && c->head_dim != 128)) {
    return noalloc_fail(FT_ERR_INVALID, "the cache needs 1 to 32767 layers, pages, 1 to 8192 key heads and head_dim 64 or 128 (got %d, %d, %d, %d)",
                        c->layers, c->pages, c->kv_heads, c->head_dim);
  }
  if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0) {
    return noalloc_fail(FT_ERR_INVALID, "page_size must be a power of two from 8 to 256 (got %d)", c->page_size);
  }
  const long long d = c->head_dim;
  const bool by_token = c->token_stride == c->kv_heads * d && c->head_stride == d;
  const bool by_head = c->token_stride == d && c->head_stride == c->page_size * d;
  if (!by_token && !by_head && !(c->kv_heads == 1 && c->token_stride == d)) {
    return noalloc_fail(FT_ERR_INVALID, "a page must be dense, by token (strides %lld, %lld) or by head (%lld, %lld)", c->kv_heads * d, d, d,
                        c->page_size * d);
  }
  if (!aligned16(c->k) || !aligned16(c->v) || c->page_stride % 8 != 0 || c->layer_stride % 8 != 0 || c->page_stride < c->page_size * c->kv_heads * d ||
      c->layer_stride < 0) {
    return noalloc_fail(FT_ERR_INVALID, "K and V must be 16-byte aligned, with page and layer strides that are multiples of 8 elements, and pages must not overlap");
  }
  // accept moves rows of all layers at once
  if (blocks_meet(c->page_stride, c->pages, c->layer_stride, c->layers, c->page_size * c->kv_heads * d)) {
    return noalloc_fail(FT_ERR_INVALID, "the pages of different layers must not share memory (layer stride %lld, page stride %lld)", c->layer_stride,
                        c->page_stride);
  }
  return FT_OK;
}

// Calls that write rows of K and rows of V at the same time.
int check_two_slabs(const ft_kv_cache* c) {
  const int rc = check_cache(c);
  if (rc == FT_OK && c->k == c->v) return noalloc_fail(FT_ERR_INVALID, "K and V of the cache are the same memory: only reading and copying pages work there");
  return rc;
}

int check_scale(float scale) {
  if (!(scale >= 0.0f) || !std::isfinite(kLog2E * scale)) {  // the exponents are in units of log2(e) * scale
    return noalloc_fail(FT_ERR_INVALID, "scale must be positive and below 2.3e38 (0: 1 / sqrt(head_dim))");
  }
  return FT_OK;
}

// The current device has to be an sm_100; its SM count, asked for once per device.
int check_device(int* sm_count) {
  static std::atomic<int> known[64];
  int device = 0;
  SERVE_CUDA(cudaGetDevice(&device));
  int count = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (count == 0) {
    int major = 0;
    SERVE_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
    if (major != 10) return noalloc_fail(FT_ERR_UNSUPPORTED, "this library needs an sm_100 GPU (found compute capability %d)", major);
    SERVE_CUDA(cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device));
    if (device < 64) known[device].store(count, std::memory_order_relaxed);
  }
  if (sm_count != nullptr) *sm_count = count;
  return FT_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A 16-bit tensor, dims and boxes innermost first, strides in elements from the second dimension on; 128-byte swizzle, zeros
// outside.  The dimensions that hold one element only may come with any stride.
int make_map(CUtensorMap* map, int dtype, const void* base, int rank, const long long* dims, const long long* strides, const int* boxes) {
  static std::atomic<EncodeTiledFn> known{nullptr};
  EncodeTiledFn encode = known.load(std::memory_order_relaxed);
  if (encode == nullptr) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult query;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &query) != cudaSuccess || query != cudaDriverEntryPointSuccess) {
      return noalloc_fail(FT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    }
    encode = reinterpret_cast<EncodeTiledFn>(sym);
    known.store(encode, std::memory_order_relaxed);
  }
  cuuint64_t d[5], s[4];
  cuuint32_t box[5], step[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    box[i] = static_cast<cuuint32_t>(boxes[i]);
    step[i] = 1;
    if (i > 0) s[i - 1] = static_cast<cuuint64_t>(dims[i] > 1 ? strides[i - 1] : dims[0]) * 2;
  }
  const CUresult r = encode(map, dtype == FT_SRC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank),
                            const_cast<void*>(base), d, s, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return noalloc_fail(FT_ERR_INVALID, "the strides or sizes of a tensor are outside what the copy engine takes (CUresult %d)", static_cast<int>(r));
  }
  return FT_OK;
}

int make_query_map(CUtensorMap* map, int dtype, const ft_rows& q, int tokens, int kv_heads, int head_dim) {
  const int group = q.heads / kv_heads;
  const long long dims[4] = {head_dim, group, kv_heads, tokens}, strides[3] = {q.head_stride, group * q.head_stride, q.token_stride};
  const int boxes[4] = {64, group, 1, 128 / group};
  return make_map(map, dtype, q.data, 4, dims, strides, boxes);
}

}  // namespace

struct ft_rotary_handle {
  ft_rotary_options options{};
  double* turns = nullptr;  // device: frequencies in turns per position
};

struct ft_page_pool {
  int page_size = 0;
  std::vector<int> users;      // per page: sequences that hold it
  std::vector<int> free_list;  // a heap, lowest page on top
  struct Sequence {
    bool used = false;
    int length = 0;
    std::vector<int> pages;
  };
  std::vector<Sequence> sequences;

  Sequence* find(int id) { return id >= 0 && id < static_cast<int>(sequences.size()) && sequences[id].used ? &sequences[id] : nullptr; }
  int take() {
    std::pop_heap(free_list.begin(), free_list.end(), std::greater<int>());
    const int page = free_list.back();
    free_list.pop_back();
    users[page] = 1;
    return page;
  }
  void drop(int page) {
    if (--users[page] == 0) {
      free_list.push_back(page);  // capacity for every page is reserved at creation
      std::push_heap(free_list.begin(), free_list.end(), std::greater<int>());
    }
  }
};

extern "C" {

// ---- rotary positions -----------------------------------------------------------

void ft_rotary_options_default(ft_rotary_options* o, int head_dim) {
  if (o == nullptr) return;
  std::memset(o, 0, sizeof(*o));
  o->head_dim = head_dim;
  o->rotary_dim = head_dim;
  o->scaling = FT_ROTARY_PLAIN;
  o->base = 10000.0;
  o->factor = 1.0;
  o->low = 1.0;
  o->high = 4.0;
  o->magnitude = 1.0;
}

int ft_rotary_frequencies(const ft_rotary_options* o, double* out) {
  if (o == nullptr || out == nullptr) return noalloc_fail(FT_ERR_INVALID, "null options or output pointer");
  if (o->head_dim <= 0 || o->head_dim > 256 || o->head_dim % 16 != 0 || o->rotary_dim <= 0 || o->rotary_dim > o->head_dim || o->rotary_dim % 16 != 0) {
    return noalloc_fail(FT_ERR_INVALID, "head_dim (at most 256) and rotary_dim (at most head_dim) must be positive multiples of 16 (got %d, %d)",
                        o->head_dim, o->rotary_dim);
  }
  if (!(o->base > 0.0) || !std::isfinite(o->base) || !(o->factor > 0.0) || !std::isfinite(o->factor) || !std::isfinite(static_cast<float>(o->magnitude))) {
    return noalloc_fail(FT_ERR_INVALID, "base and factor must be positive, magnitude finite in 32 bits");
  }
  if (o->scaling < FT_ROTARY_PLAIN || o->scaling > FT_ROTARY_BY_PARTS) return noalloc_fail(FT_ERR_INVALID, "unknown scaling %d", o->scaling);
  if (o->scaling == FT_ROTARY_BY_PARTS &&
      (!(o->original_length > 0.0) || !std::isfinite(o->original_length) || !(o->high > o->low) || !std::isfinite(o->low) || !std::isfinite(o->high))) {
    return noalloc_fail(FT_ERR_INVALID, "scaling by parts needs original_length > 0 and high > low");
  }
  const double two_pi = 6.283185307179586476925286766559;
  const double dim = o->rotary_dim;
  const double base = o->scaling == FT_ROTARY_BASE ? o->base * std::pow(o->factor, dim / (dim - 2.0)) : o->base;
  for (int i = 0; i < o->rotary_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / dim);
    if (o->scaling == FT_ROTARY_LINEAR) f /= o->factor;
    if (o->scaling == FT_ROTARY_BY_PARTS) {
      const double keep = std::min(1.0, std::max(0.0, (o->original_length * f / two_pi - o->low) / (o->high - o->low)));
      f *= keep + (1.0 - keep) / o->factor;
    }
    if (!std::isfinite(f) || !std::isfinite(base)) return noalloc_fail(FT_ERR_INVALID, "base and factor give frequencies that are not finite");
    out[i] = f;
  }
  return FT_OK;
}

int ft_rotary_destroy(ft_rotary_handle* h) {
  if (h == nullptr) return FT_OK;
  cudaFree(h->turns);
  delete h;
  return FT_OK;
}

int ft_rotary_prepare(ft_rotary_handle** handle, const ft_rotary_options* options, void* stream) {
  if (handle == nullptr) return noalloc_fail(FT_ERR_INVALID, "null handle pointer");
  *handle = nullptr;
  double turns[128];
  int rc = ft_rotary_frequencies(options, turns);
  if (rc == FT_OK) rc = check_device(nullptr);
  if (rc != FT_OK) return rc;
  const int count = options->rotary_dim / 2;
  for (int i = 0; i < count; ++i) turns[i] /= 6.283185307179586476925286766559;
  ft_rotary_handle* h = new (std::nothrow) ft_rotary_handle();
  if (h == nullptr) return noalloc_fail(FT_ERR_INVALID, "out of host memory");
  h->options = *options;
  cudaError_t err = cudaMalloc(reinterpret_cast<void**>(&h->turns), count * sizeof(double));
  // pageable host memory: the copy has left `turns` when the call returns; the wait makes the handle valid on every stream
  if (err == cudaSuccess) err = cudaMemcpyAsync(h->turns, turns, count * sizeof(double), cudaMemcpyHostToDevice, static_cast<cudaStream_t>(stream));
  if (err == cudaSuccess) err = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) {
    ft_rotary_destroy(h);
    return noalloc_fail(FT_ERR_CUDA, "preparing the rotary frequencies failed: %s", cudaGetErrorString(err));
  }
  *handle = h;
  return FT_OK;
}

// Rows of a block and blocks of a launch are counted in 31 bits.
constexpr int kMaxRows = 1 << 30, kMaxHeads = 1 << 20;

static void use_rotary(RotaryParams* p, const ft_rotary_handle* h) {
  p->turns = h->turns;
  p->rotary_dim = h->options.rotary_dim;
  p->head_dim = h->options.head_dim;
  p->interleaved = h->options.interleaved != 0;
  p->magnitude = static_cast<float>(h->options.magnitude);
}

int ft_rotary_run(const ft_rotary_handle* h, const ft_rows* q, const ft_rows* q_out, const ft_rows* k, const ft_rows* k_out, const long long* positions,
                  int tokens, int dtype, int inverse, void* stream) {
  if (h == nullptr || positions == nullptr) return noalloc_fail(FT_ERR_INVALID, "null handle or positions");
  if (tokens < 0 || tokens > kMaxRows) return noalloc_fail(FT_ERR_INVALID, "negative token count, or more than 2^30 tokens");
  if (q == nullptr || q->heads <= 0 || (k != nullptr && k->heads <= 0)) return noalloc_fail(FT_ERR_INVALID, "q needs at least one head, and k if given");
  if (q->heads > kMaxHeads || (k != nullptr && k->heads > kMaxHeads)) return noalloc_fail(FT_ERR_INVALID, "q and k have at most %d heads", kMaxHeads);
  int rc = check_dtype(dtype);
  if (rc == FT_OK) rc = check_rows(q, "q", q->heads);
  if (rc == FT_OK) rc = check_rows(q_out, "q_out", q->heads);
  if (rc == FT_OK && k != nullptr) rc = check_rows(k, "k", k->heads);
  if (rc == FT_OK && k != nullptr) rc = check_rows(k_out, "k_out", k->heads);
  if (rc == FT_OK) rc = check_output(q_out, "q_out", tokens, h->options.head_dim, q);
  if (rc == FT_OK && k != nullptr) rc = check_output(k_out, "k_out", tokens, h->options.head_dim, k);
  if (rc == FT_OK && k != nullptr && tokens > 0 && q_out->data == k_out->data) rc = noalloc_fail(FT_ERR_INVALID, "q_out and k_out share memory");
  if (rc != FT_OK) return rc;
  RotaryParams p{};
  use_rotary(&p, h);
  p.q = to_rows(q);
  p.q_out = to_rows(q_out);
  p.q_heads = q->heads;
  if (k != nullptr) {
    p.k = to_rows(k);
    p.k_out = to_rows(k_out);
    p.k_heads = k->heads;
  }
  p.positions = positions;
  p.tokens = tokens;
  p.inverse = inverse != 0;
  SERVE_CUDA(launch_rotary(p, dtype, static_cast<cudaStream_t>(stream)));
  return FT_OK;
}

// ---- paged key/value cache -------------------------------------------------------

int ft_kv_cache_append(const ft_kv_cache* cache, int layer, const ft_rows* k, const ft_rows* v, const long long* slots, int tokens,
                       const ft_rotary_handle* rotary, const long long* positions, const ft_rows* q, const ft_rows* q_out, void* stream) {
  int rc = check_two_slabs(cache);
  if (rc != FT_OK) return rc;
  if (layer < 0 || layer >= cache->layers) return noalloc_fail(FT_ERR_INVALID, "layer %d is outside the cache's %d", layer, cache->layers);
  if (slots == nullptr) return noalloc_fail(FT_ERR_INVALID, "null slots");
  if (tokens < 0 || tokens > kMaxRows) return noalloc_fail(FT_ERR_INVALID, "negative token count, or more than 2^30 tokens");
  rc = check_rows(k, "k", cache->kv_heads);
  if (rc == FT_OK) rc = check_rows(v, "v", cache->kv_heads);
  if (rc != FT_OK) return rc;
  if (rotary == nullptr && q != nullptr) return noalloc_fail(FT_ERR_INVALID, "q is only rotated with a rotary handle");
  if (rotary != nullptr && positions == nullptr) return noalloc_fail(FT_ERR_INVALID, "null positions");
  if (rotary != nullptr && rotary->options.head_dim != cache->head_dim) {
    return noalloc_fail(FT_ERR_INVALID, "the rotary handle is for head_dim %d, the cache has %d", rotary->options.head_dim, cache->head_dim);
  }
  RotaryParams p{};
  p.head_dim = cache->head_dim;
  if (rotary != nullptr) use_rotary(&p, rotary);
  if (q != nullptr) {
    if (q->heads <= 0 || q->heads > kMaxHeads) return noalloc_fail(FT_ERR_INVALID, "q needs 1 to %d heads", kMaxHeads);
    rc = check_rows(q, "q", q->heads);
    if (rc == FT_OK) rc = check_rows(q_out, "q_out", q->heads);
    if (rc == FT_OK) rc = check_output(q_out, "q_out", tokens, cache->head_dim, q);
    if (rc != FT_OK) return rc;
    p.q = to_rows(q);
    p.q_out = to_rows(q_out);
    p.q_heads = q->heads;
  }
  p.k = to_rows(k);
  p.v = to_rows(v);
  p.k_heads = p.v_heads = cache->kv_heads;
  p.positions = positions;
  p.slots = slots;
  p.k_cache = static_cast<uint16_t*>(cache->k) + layer * cache->layer_stride;
  p.v_cache = static_cast<uint16_t*>(cache->v) + layer * cache->layer_stride;
  p.page_stride = cache->page_stride;
  p.cache_token_stride = cache->token_stride;
  p.cache_head_stride = cache->head_stride;
  while ((1 << p.page_shift) < cache->page_size) ++p.page_shift;
  p.slot_count = static_cast<long long>(cache->pages) * cache->page_size;
  p.tokens = tokens;
  SERVE_CUDA(launch_rotary(p, cache->dtype, static_cast<cudaStream_t>(stream)));
  return FT_OK;
}

int ft_kv_cache_copy_pages(const ft_kv_cache* cache, const int* sources, const int* targets, int count, void* stream) {
  int rc = check_cache(cache);
  if (rc != FT_OK) return rc;
  if (count < 0 || (count > 0 && (sources == nullptr || targets == nullptr))) {
    return noalloc_fail(FT_ERR_INVALID, "copying pages needs pairs with sources and targets (got %d)", count);
  }
  if (count > copy_pages_most(cache->page_size * cache->kv_heads * cache->head_dim)) {  // blocks are counted in 31 bits
    return noalloc_fail(FT_ERR_INVALID, "%d pages at once are too many: at most %d of this size", count,
                        copy_pages_most(cache->page_size * cache->kv_heads * cache->head_dim));
  }
  CopyPagesParams p{};
  p.k = static_cast<uint16_t*>(cache->k);
  p.v = static_cast<uint16_t*>(cache->v);
  p.layer_stride = cache->layer_stride;
  p.page_stride = cache->page_stride;
  p.layers = cache->layers;
  p.pages = cache->pages;
  p.page_elements = cache->page_size * cache->kv_heads * cache->head_dim;
  p.count = count;
  p.sources = sources;
  p.targets = targets;
  SERVE_CUDA(launch_copy_pages(p, static_cast<cudaStream_t>(stream)));
  return FT_OK;
}

int ft_kv_cache_accept(const ft_kv_cache* cache, const int* page_table, int table_pages, int table_stride, const int* lengths,
                       const int* drafted_offsets, const int* accepted, const int* accepted_offsets, int batch, int* new_lengths, void* stream) {
  int rc = check_two_slabs(cache);
  if (rc != FT_OK) return rc;
  if (batch < 0 || table_pages <= 0 || table_stride < table_pages) {
    return noalloc_fail(FT_ERR_INVALID, "batch must not be negative, the page table needs columns and a stride that holds them");
  }
  if (page_table == nullptr || lengths == nullptr || drafted_offsets == nullptr || accepted == nullptr || accepted_offsets == nullptr ||
      new_lengths == nullptr) {
    return noalloc_fail(FT_ERR_INVALID, "null page table, lengths, offsets or accepted tokens");
  }
  if (lengths == new_lengths) return noalloc_fail(FT_ERR_INVALID, "new_lengths must not be the lengths array");
  AcceptParams p{};
  p.k = static_cast<uint16_t*>(cache->k);
  p.v = static_cast<uint16_t*>(cache->v);
  p.layer_stride = cache->layer_stride;
  p.page_stride = cache->page_stride;
  p.token_stride = cache->token_stride;
  p.head_stride = cache->head_stride;
  p.layers = cache->layers;
  p.pages = cache->pages;
  p.page_size = cache->page_size;
  p.kv_heads = cache->kv_heads;
  p.head_dim = cache->head_dim;
  p.page_table = page_table;
  p.table_pages = table_pages;
  p.table_stride = table_stride;
  p.lengths = lengths;
  p.drafted_offsets = drafted_offsets;
  p.accepted = accepted;
  p.accepted_offsets = accepted_offsets;
  p.batch = batch;
  p.new_lengths = new_lengths;
  SERVE_CUDA(launch_accept(p, static_cast<cudaStream_t>(stream)));
  return FT_OK;
}

// ---- page pool -------------------------------------------------------------------

int ft_page_pool_create(ft_page_pool** pool, int pages, int page_size) {
  if (pool == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool pointer");
  *pool = nullptr;
  if (pages <= 0 || page_size <= 0) return noalloc_fail(FT_ERR_INVALID, "a pool needs pages and a page size");
  try {
    ft_page_pool* p = new ft_page_pool();
    *pool = p;
    p->page_size = page_size;
    p->users.assign(pages, 0);
    p->free_list.resize(pages);
    for (int i = 0; i < pages; ++i) p->free_list[i] = i;  // ascending: a heap already
  } catch (const std::bad_alloc&) {
    delete *pool;
    *pool = nullptr;
    return noalloc_fail(FT_ERR_INVALID, "out of host memory");
  }
  return FT_OK;
}

int ft_page_pool_destroy(ft_page_pool* pool) {
  delete pool;
  return FT_OK;
}

int ft_page_pool_free_pages(const ft_page_pool* pool) {
  if (pool == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool");
  return static_cast<int>(pool->free_list.size());
}

int ft_page_pool_new_sequence(ft_page_pool* pool, int* sequence) {
  if (pool == nullptr || sequence == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool or sequence pointer");
  auto& all = pool->sequences;
  size_t id = 0;
  while (id < all.size() && all[id].used) ++id;
  try {
    if (id == all.size()) all.emplace_back();
  } catch (const std::bad_alloc&) {
    return noalloc_fail(FT_ERR_INVALID, "out of host memory");
  }
  all[id].used = true;
  all[id].length = 0;
  all[id].pages.clear();
  *sequence = static_cast<int>(id);
  return FT_OK;
}

int ft_page_pool_fork(ft_page_pool* pool, int sequence, int* child) {
  if (pool == nullptr || child == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool or sequence pointer");
  if (pool->find(sequence) == nullptr) return noalloc_fail(FT_ERR_INVALID, "no sequence %d", sequence);
  int id = 0;
  const int rc = ft_page_pool_new_sequence(pool, &id);
  if (rc != FT_OK) return rc;
  ft_page_pool::Sequence& parent = pool->sequences[sequence];
  ft_page_pool::Sequence& made = pool->sequences[id];
  try {
    made.pages = parent.pages;
  } catch (const std::bad_alloc&) {
    made.used = false;
    return noalloc_fail(FT_ERR_INVALID, "out of host memory");
  }
  made.length = parent.length;
  for (int page : made.pages) ++pool->users[page];
  *child = id;
  return FT_OK;
}

int ft_page_pool_free(ft_page_pool* pool, int sequence) {
  if (pool == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool");
  ft_page_pool::Sequence* s = pool->find(sequence);
  if (s == nullptr) return noalloc_fail(FT_ERR_INVALID, "no sequence %d", sequence);
  for (int page : s->pages) pool->drop(page);
  s->pages.clear();
  s->length = 0;
  s->used = false;
  return FT_OK;
}

int ft_page_pool_extend(ft_page_pool* pool, int sequence, int tokens, int* source, int* target) {
  if (pool == nullptr || source == nullptr || target == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool or pair pointer");
  *source = *target = -1;
  ft_page_pool::Sequence* s = pool->find(sequence);
  if (s == nullptr) return noalloc_fail(FT_ERR_INVALID, "no sequence %d", sequence);
  if (tokens < 0 || tokens > INT32_MAX - s->length) return noalloc_fail(FT_ERR_INVALID, "a sequence cannot grow by %d tokens", tokens);
  if (tokens == 0) return FT_OK;
  const int size = pool->page_size, length = s->length + tokens;
  const size_t held = s->pages.size(), need = (static_cast<size_t>(length) + size - 1) / size;
  // the page that the first new token goes to is written: it must be this sequence's alone
  const bool copy = s->length % size != 0 && pool->users[s->pages[s->length / size]] > 1;
  const size_t take = need - held + (copy ? 1 : 0);
  if (take > pool->free_list.size()) {
    return noalloc_fail(FT_ERR_INVALID, "the pool has %zu free pages, %zu are needed", pool->free_list.size(), take);
  }
  try {
    s->pages.reserve(need);
  } catch (const std::bad_alloc&) {
    return noalloc_fail(FT_ERR_INVALID, "out of host memory");
  }
  if (copy) {
    int& last = s->pages[s->length / size];
    *source = last;
    *target = pool->take();
    pool->drop(last);
    last = *target;
  }
  while (s->pages.size() < need) s->pages.push_back(pool->take());
  s->length = length;
  return FT_OK;
}

int ft_page_pool_truncate(ft_page_pool* pool, int sequence, int length) {
  if (pool == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool");
  ft_page_pool::Sequence* s = pool->find(sequence);
  if (s == nullptr) return noalloc_fail(FT_ERR_INVALID, "no sequence %d", sequence);
  if (length < 0 || length > s->length) return noalloc_fail(FT_ERR_INVALID, "sequence %d holds %d tokens, it cannot be cut to %d", sequence, s->length, length);
  const size_t need = (static_cast<size_t>(length) + pool->page_size - 1) / pool->page_size;
  while (s->pages.size() > need) {
    pool->drop(s->pages.back());
    s->pages.pop_back();
  }
  s->length = length;
  return FT_OK;
}

int ft_page_pool_length(const ft_page_pool* pool, int sequence) {
  if (pool == nullptr) return noalloc_fail(FT_ERR_INVALID, "null pool");
  const ft_page_pool::Sequence* s = const_cast<ft_page_pool*>(pool)->find(sequence);
  if (s == nullptr) return noalloc_fail(FT_ERR_INVALID, "no sequence %d", sequence);
  return s->length;
}

int ft_page_pool_pages(const ft_page_pool* pool, int sequence, int* out, int capacity) {
  if (pool == nullptr || (out == nullptr && capacity > 0) || capacity < 0) return noalloc_fail(FT_ERR_INVALID, "null pool or page array");
  const ft_page_pool::Sequence* s = const_cast<ft_page_pool*>(pool)->find(sequence);
  if (s == nullptr) return noalloc_fail(FT_ERR_INVALID, "no sequence %d", sequence);
  const int count = static_cast<int>(s->pages.size());
  std::copy(s->pages.begin(), s->pages.begin() + std::min(count, capacity), out);
  return count;
}

int ft_page_pool_compact(ft_page_pool* pool, int* sources, int* targets, int capacity, int* count) {
  if (pool == nullptr || count == nullptr || capacity < 0 || (capacity > 0 && (sources == nullptr || targets == nullptr))) {
    return noalloc_fail(FT_ERR_INVALID, "null pool, pairs or count");
  }
  *count = 0;
  try {
    std::vector<int> moved(pool->users.size(), -1);
    std::vector<int> free_after;
    free_after.reserve(pool->users.size());
    int low = 0, high = static_cast<int>(pool->users.size()) - 1, n = 0;
    while (n < capacity) {
      while (low < high && pool->users[low] > 0) ++low;
      while (low < high && pool->users[high] == 0) --high;
      if (low >= high) break;
      sources[n] = high;
      targets[n++] = low;
      moved[high] = low;
      pool->users[low] = pool->users[high];
      pool->users[high] = 0;
    }
    for (auto& s : pool->sequences) {
      for (int& page : s.pages) {
        if (moved[page] >= 0) page = moved[page];
      }
    }
    pool->free_list.clear();
    for (int i = 0; i < static_cast<int>(pool->users.size()); ++i) {
      if (pool->users[i] == 0) pool->free_list.push_back(i);
    }
    *count = n;
  } catch (const std::bad_alloc&) {
    return noalloc_fail(FT_ERR_INVALID, "out of host memory");
  }
  return FT_OK;
}

// ---- attention -------------------------------------------------------------------

size_t ft_attention_workspace(void) {
  int sm_count = 0;
  return check_device(&sm_count) == FT_OK ? serve_attention_workspace(sm_count) : 0;
}

constexpr int kMaxQueries = 1 << 30;  // sums of a few of them stay inside 32 bits
// A warp that has nothing to do for a row tile waits while the others go through its keys, and waits give up after 4
// seconds: 2^20 key tiles take 2 to 3.
constexpr int kMaxKeys = 1 << 27;

static int check_heads(int heads, int kv_heads) {
  if (kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 || heads / kv_heads > 128) {
    return noalloc_fail(FT_ERR_INVALID, "query heads (%d) must be 1 to 128 times the key heads (%d)", heads, kv_heads);
  }
  return FT_OK;
}

static int check_workspace(const void* workspace, size_t bytes, const int* status) {
  if (workspace == nullptr || bytes == 0 || !aligned16(workspace)) return noalloc_fail(FT_ERR_INVALID, "the workspace must be there and 16-byte aligned");
  if (status == nullptr) return noalloc_fail(FT_ERR_INVALID, "null status");
  return FT_OK;
}

// What both calls share: the rows of q and out, the launch.
static int attention_run(ServeAttentionParams& p, const ft_rows& q, const ft_rows& out, const CUtensorMap& k_map, const CUtensorMap& v_map, int dtype,
                         long long most_keys, float scale, void* workspace, size_t workspace_bytes, int* status, int sm_count, void* stream) {
  if (workspace_bytes < serve_attention_workspace(sm_count)) {
    return noalloc_fail(FT_ERR_INVALID, "the workspace holds %zu bytes, ft_attention_workspace() says %zu", workspace_bytes,
                        serve_attention_workspace(sm_count));
  }
  CUtensorMap q_map;
  const int rc = make_query_map(&q_map, dtype, q, p.query_tokens, p.kv_heads, p.head_dim);
  if (rc != FT_OK) return rc;
  p.out = static_cast<uint16_t*>(out.data);
  p.out_token_stride = out.token_stride;
  p.out_head_stride = out.head_stride;
  p.heads = q.heads;
  p.group = q.heads / p.kv_heads;
  p.tokens_per_tile = 128 / p.group;
  p.scale_log2 = kLog2E * (scale != 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(p.head_dim)));
  // an upper bound on the units of work (serving_schedule.h), which are numbered in 31 bits
  const long long row_tiles = static_cast<long long>(p.query_tokens) / p.tokens_per_tile + p.batch;
  const bool may_pass = row_tiles > INT32_MAX / 8 || row_tiles * p.kv_heads > INT32_MAX / (most_keys / 128 + 8);
  // Several packed sequences have all keys between them, so the bound can be far off: the device counts.
  p.count_units = may_pass && p.page_table == nullptr && p.batch > 1;
  if (row_tiles > INT32_MAX / 8 || (may_pass && p.count_units == 0)) {
    return noalloc_fail(FT_ERR_INVALID, "the call is too large: %lld tiles of query rows for %d key heads over up to %lld keys", row_tiles, p.kv_heads, most_keys);
  }
  p.workspace = workspace;
  p.status = status;
  // Two tiles of rows that go through the keys together halve what is read of K and V.  That needs sequences of more than
  // one tile, and enough key tiles for every SM; below that the finer items fill the SMs better.  (Only sizes that the
  // host knows go into this: averages over the sequences, and the most keys there can be.)  B200, 32 heads of 128 on 8: trees
  // of 64 and 31 tokens over 131072 and 65001 keys 223 us split, 194 us in pairs; a prompt of 200 tokens 11.3 and 16.4 us; 64
  // single tokens over up to 8060 keys 69 and 89 us.
  const long long tiles = (static_cast<long long>(p.query_tokens) + p.tokens_per_tile - 1) / p.tokens_per_tile;
  const long long keys = p.page_table != nullptr ? most_keys : most_keys / p.batch;
  const bool pairs = tiles > p.batch && tiles * p.kv_heads * (keys / 128 + 1) >= 4ll * sm_count;
  SERVE_CUDA(launch_serve_attention(q_map, k_map, v_map, p, dtype, !pairs, sm_count, static_cast<cudaStream_t>(stream)));
  return FT_OK;
}

int ft_prompt_attention_run(const ft_prompt_attention_args* a, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (a == nullptr) return noalloc_fail(FT_ERR_INVALID, "null arguments");
  int rc = check_workspace(workspace, workspace_bytes, status);
  if (rc == FT_OK) rc = check_heads(a->q.heads, a->k.heads);
  if (rc == FT_OK) rc = check_dtype(a->dtype);
  if (rc == FT_OK) rc = check_scale(a->scale);
  if (rc != FT_OK) return rc;
  if (a->head_dim != 64 && a->head_dim != 128) return noalloc_fail(FT_ERR_INVALID, "head_dim must be 64 or 128 (got %d)", a->head_dim);
  if (a->batch < 0 || a->query_tokens < 0 || a->key_tokens < 0 || a->query_tokens > kMaxQueries || a->key_tokens > kMaxKeys) {
    return noalloc_fail(FT_ERR_INVALID, "negative batch or token count, more than 2^30 queries or more than 2^27 keys");
  }
  if (a->batch == 0 || a->query_tokens == 0) return FT_OK;
  if (a->q_offsets == nullptr) return noalloc_fail(FT_ERR_INVALID, "null q_offsets");
  rc = check_rows(&a->q, "q", a->q.heads);
  if (rc == FT_OK) rc = check_rows(&a->out, "out", a->q.heads);
  if (rc == FT_OK) rc = check_apart(&a->q, "q", a->query_tokens, a->head_dim);
  if (rc == FT_OK) rc = check_output(&a->out, "out", a->query_tokens, a->head_dim, nullptr);
  if (rc == FT_OK && a->key_tokens > 0) {
    rc = check_rows(&a->k, "k", a->k.heads);
    if (rc == FT_OK) rc = check_rows(&a->v, "v", a->k.heads);
    if (rc == FT_OK) rc = check_apart(&a->k, "k", a->key_tokens, a->head_dim);
    if (rc == FT_OK) rc = check_apart(&a->v, "v", a->key_tokens, a->head_dim);
  }
  int sm_count = 0;
  if (rc == FT_OK) rc = check_device(&sm_count);
  if (rc != FT_OK) return rc;
  CUtensorMap maps[2];
  const ft_rows* kv[2] = {&a->k, &a->v};
  for (int i = 0; i < 2; ++i) {
    // without any key nothing is read: the map then only has to be one
    const ft_rows& rows = a->key_tokens > 0 ? *kv[i] : a->q;
    const long long dims[3] = {a->head_dim, a->key_tokens > 0 ? a->k.heads : 1, std::max(a->key_tokens, 1)}, strides[2] = {rows.head_stride, rows.token_stride};
    const int boxes[3] = {64, 1, 128};
    rc = make_map(&maps[i], a->dtype, rows.data, 3, dims, strides, boxes);
    if (rc != FT_OK) return rc;
  }
  ServeAttentionParams p{};
  p.lse = a->lse;
  p.q_offsets = a->q_offsets;
  p.k_offsets = a->k_offsets != nullptr ? a->k_offsets : a->q_offsets;
  p.batch = a->batch;
  p.query_tokens = a->query_tokens;
  p.key_tokens = a->key_tokens;
  p.kv_heads = a->k.heads;
  p.head_dim = a->head_dim;
  p.causal = a->causal != 0;
  return attention_run(p, a->q, a->out, maps[0], maps[1], a->dtype, a->key_tokens, a->scale, workspace, workspace_bytes, status, sm_count, stream);
}

int ft_tree_attention_run(const ft_kv_cache* cache, const ft_tree_attention_args* a, void* workspace, size_t workspace_bytes, int* status,
                          void* stream) {
  if (a == nullptr) return noalloc_fail(FT_ERR_INVALID, "null arguments");
  int rc = check_cache(cache);
  if (rc == FT_OK) rc = check_workspace(workspace, workspace_bytes, status);
  if (rc == FT_OK) rc = check_heads(a->q.heads, cache->kv_heads);
  if (rc == FT_OK) rc = check_scale(a->scale);
  if (rc != FT_OK) return rc;
  if (a->layer < 0 || a->layer >= cache->layers) return noalloc_fail(FT_ERR_INVALID, "layer %d is outside the cache's %d", a->layer, cache->layers);
  if (a->batch < 0 || a->query_tokens < 0 || a->query_tokens > kMaxQueries) {
    return noalloc_fail(FT_ERR_INVALID, "negative batch or token count, or more than 2^30 queries");
  }
  if (a->table_pages <= 0 || a->table_stride < a->table_pages || a->table_pages > kMaxKeys / cache->page_size) {
    return noalloc_fail(FT_ERR_INVALID, "the page table needs columns (at most 2^27 tokens) and a stride that holds them (got %d, %d)", a->table_pages,
                        a->table_stride);
  }
  if (a->mask != nullptr && (a->mask_words <= 0 || a->mask_stride < a->mask_words)) {
    return noalloc_fail(FT_ERR_INVALID, "the mask needs words and a stride that holds them (got %d, %d)", a->mask_words, a->mask_stride);
  }
  if (a->batch == 0 || a->query_tokens == 0) return FT_OK;
  if (a->q_offsets == nullptr || a->page_table == nullptr || a->lengths == nullptr) return noalloc_fail(FT_ERR_INVALID, "null q_offsets, page table or lengths");
  rc = check_rows(&a->q, "q", a->q.heads);
  if (rc == FT_OK) rc = check_rows(&a->out, "out", a->q.heads);
  if (rc == FT_OK) rc = check_apart(&a->q, "q", a->query_tokens, cache->head_dim);
  if (rc == FT_OK) rc = check_output(&a->out, "out", a->query_tokens, cache->head_dim, nullptr);
  if (rc != FT_OK) return rc;
  // The copy engine sees groups of 8 tokens, numbered over all pages.
  const long long page_groups = cache->page_stride / (8 * cache->token_stride);
  const long long groups = (cache->pages - 1) * page_groups + cache->page_size / 8;
  if (cache->page_stride % (8 * cache->token_stride) != 0 || (cache->pages + 1) * page_groups > INT32_MAX) {
    return noalloc_fail(FT_ERR_INVALID, "the page stride (%lld) must be a multiple of that of 8 tokens (%lld), with fewer than 2^31 of them in the cache",
                        cache->page_stride, 8 * cache->token_stride);
  }
  int sm_count = 0;
  rc = check_device(&sm_count);
  if (rc != FT_OK) return rc;
  CUtensorMap maps[2];
  void* const kv[2] = {cache->k, cache->v};
  for (int i = 0; i < 2; ++i) {
    const long long dims[5] = {64, 8, cache->head_dim / 64, groups, cache->kv_heads};
    const long long strides[4] = {cache->token_stride, 64, 8 * cache->token_stride, cache->head_stride};
    const int boxes[5] = {64, 8, cache->head_dim / 64, std::min(cache->page_size, 128) / 8, 1};
    rc = make_map(&maps[i], cache->dtype, static_cast<const uint16_t*>(kv[i]) + a->layer * cache->layer_stride, 5, dims, strides, boxes);
    if (rc != FT_OK) return rc;
  }
  ServeAttentionParams p{};
  p.lse = a->lse;
  p.q_offsets = a->q_offsets;
  p.page_table = a->page_table;
  p.lengths = a->lengths;
  p.mask = a->mask;
  p.mask_words = a->mask_words;
  p.mask_stride = a->mask_stride;
  p.batch = a->batch;
  p.query_tokens = a->query_tokens;
  p.kv_heads = cache->kv_heads;
  p.head_dim = cache->head_dim;
  p.causal = 1;
  p.page_size = cache->page_size;
  p.page_groups = static_cast<int>(page_groups);
  p.pages = cache->pages;
  p.table_pages = a->table_pages;
  p.table_stride = a->table_stride;
  return attention_run(p, a->q, a->out, maps[0], maps[1], cache->dtype, static_cast<long long>(a->table_pages) * cache->page_size, a->scale, workspace,
                       workspace_bytes, status, sm_count, stream);
}

int ft_tree_mask(const int* parents, int nodes, uint32_t* mask, int words) {
  if (nodes < 0 || words < 0 || (nodes > 0 && (parents == nullptr || mask == nullptr)) || nodes > static_cast<long long>(words) * 32) {
    return noalloc_fail(FT_ERR_INVALID, "a tree of %d nodes needs parents and a mask of at least as many bits (%d words)", nodes, words);
  }
  for (int i = 0; i < nodes; ++i) {
    if (parents[i] >= i) return noalloc_fail(FT_ERR_INVALID, "node %d has the parent %d: parents come before their children", i, parents[i]);
    uint32_t* row = mask + static_cast<size_t>(i) * words;
    if (parents[i] >= 0) {
      std::copy(mask + static_cast<size_t>(parents[i]) * words, mask + static_cast<size_t>(parents[i] + 1) * words, row);
    } else {
      std::fill(row, row + words, 0u);
    }
    row[i / 32] |= 1u << (i % 32);
  }
  return FT_OK;
}

}  // extern "C"
