// Rotary positions and the page operations of the key/value cache: one pass over the
// data each, bound by HBM for many tokens and by launch latency for few.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "serving_kernels.h"

namespace ftg {

namespace {

__device__ __forceinline__ float2 unpack(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 unpack(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ void pack(__half2& d, float x, float y) { d = __floats2half2_rn(x, y); }
__device__ __forceinline__ void pack(__nv_bfloat162& d, float x, float y) { d = __floats2bfloat162_rn(x, y); }

template <typename T>
union Chunk {  // 16 bytes: eight elements
  uint4 raw;
  T pairs[4];
};

// Rotates, copies and scatters the rows of `tokens_per_block` tokens.  A thread takes two 16-byte chunks of a row: the
// two halves of eight pairs (or, interleaved, eight pairs outright), or two chunks that are only copied.  Sines and cosines
// are computed once per token and frequency, shared by all heads, while the first rows are on their way: the angle in
// turns is position * frequency / 2pi, formed and reduced to [-1/2, 1/2] in 64 bits (32 bits lose it beyond some ten
// thousand positions), then one sincospi in 32 bits.
// Bound by HBM for many tokens: 16384 tokens of 32 + 8 heads of 128 with the append, 403 MB, in 64 us = 6.3 TB/s (0.96 of the
// measured copy rate); of the shapes tried (128 to 512 threads, 1 to 8 tokens a block, 1 to 3 rows in flight per thread: 64
// to 100 us) many resident warps with one row each are the fastest.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p, int tokens_per_block) {
  extern __shared__ float2 turn[];  // [token in block][rotary_dim / 2]: magnitude * (cos, sin)
  const int half = p.rotary_dim / 2;
  const int first = blockIdx.x * tokens_per_block;
  const int count = min(tokens_per_block, p.tokens - first);
  const int rows = p.q_heads + p.k_heads + p.v_heads;
  const int unit = threadIdx.x;  // which two chunks of the row
  const int rotated_units = p.rotary_dim / 16;

  struct Work {
    uint16_t* dst;  // nullptr: nothing to do
    int token;      // in the block
    bool rotate;
    Chunk<T> a, b;
  };
  auto places = [&](bool rotate, int& at0, int& at1) {
    const bool halves = rotate && !p.interleaved;
    at0 = halves ? unit * 8 : unit * 16;
    at1 = halves ? at0 + half : at0 + 8;
  };
  auto load = [&](int r, Work& w) {
    w.dst = nullptr;
    if (r >= count * rows) return;
    w.token = r / rows;
    int head = r - w.token * rows;
    const long long token = first + w.token;
    const uint16_t* src;
    w.rotate = unit < rotated_units;
    if (head < p.q_heads) {
      src = p.q.data + token * p.q.token_stride + head * p.q.head_stride;
      w.dst = p.q_out.data + token * p.q_out.token_stride + head * p.q_out.head_stride;
    } else {
      head -= p.q_heads;
      const bool value = head >= p.k_heads;
      if (value) {
        head -= p.k_heads;
        w.rotate = false;
      }
      const Rows& rows_in = value ? p.v : p.k;
      src = rows_in.data + token * rows_in.token_stride + head * rows_in.head_stride;
      if (p.slots != nullptr) {
        const long long slot = p.slots[token];
        if (slot < 0 || slot >= p.slot_count) return;  // padding of the batch
        w.dst = (value ? p.v_cache : p.k_cache) + (slot >> p.page_shift) * p.page_stride + (slot & ((1 << p.page_shift) - 1)) * p.cache_token_stride +
                head * p.cache_head_stride;
      } else {
        w.dst = p.k_out.data + token * p.k_out.token_stride + head * p.k_out.head_stride;
      }
    }
    int at0, at1;
    places(w.rotate, at0, at1);
    w.a.raw = *reinterpret_cast<const uint4*>(src + at0);
    w.b.raw = *reinterpret_cast<const uint4*>(src + at1);
  };
  auto finish = [&](Work& w) {
    if (w.dst == nullptr) return;
    if (w.rotate) {
      const float2* cs = turn + w.token * half + unit * 8;
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = unpack(w.a.pairs[i]), y = unpack(w.b.pairs[i]);
          const float2 u = cs[i], v = cs[4 + i];
          pack(w.a.pairs[i], x.x * u.x - x.y * u.y, x.x * u.y + x.y * u.x);
          pack(w.b.pairs[i], y.x * v.x - y.y * v.y, y.x * v.y + y.y * v.x);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = unpack(w.a.pairs[i]), y = unpack(w.b.pairs[i]);
          const float2 u = cs[2 * i], v = cs[2 * i + 1];
          pack(w.a.pairs[i], x.x * u.x - y.x * u.y, x.y * v.x - y.y * v.y);
          pack(w.b.pairs[i], x.x * u.y + y.x * u.x, x.y * v.y + y.y * v.x);
        }
      }
    }
    int at0, at1;
    places(w.rotate, at0, at1);
    *reinterpret_cast<uint4*>(w.dst + at0) = w.a.raw;
    *reinterpret_cast<uint4*>(w.dst + at1) = w.b.raw;
  };

  Work work;
  load(threadIdx.y, work);
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < count * half; i += blockDim.x * blockDim.y) {
    const int t = i / half, f = i - t * half;
    double angle = static_cast<double>(p.positions[first + t]) * p.turns[f];
    angle -= rint(angle);
    float s, c;
    sincospif(2.0f * static_cast<float>(angle), &s, &c);
    turn[i] = make_float2(c * p.magnitude, (p.inverse ? -s : s) * p.magnitude);
  }
  __syncthreads();
  for (int r = threadIdx.y; r < count * rows;) {
    finish(work);
    r += blockDim.y;
    load(r, work);
  }
}

// Whole pages, a block for each 16 KiB piece of one page of one layer, of K or of V.
constexpr int kCopyThreads = 256, kCopyUnroll = 4;

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyPagesParams p, int pieces) {
  const int pair = blockIdx.x / pieces, piece = blockIdx.x - pair * pieces;
  const int source = p.sources[pair], target = p.targets[pair];
  if (source < 0 || source >= p.pages || target < 0 || target >= p.pages || source == target) return;
  uint16_t* base = (blockIdx.y & 1 ? p.v : p.k) + (blockIdx.y >> 1) * p.layer_stride;
  const uint4* src = reinterpret_cast<const uint4*>(base + source * p.page_stride);
  uint4* dst = reinterpret_cast<uint4*>(base + target * p.page_stride);
  const int chunks = p.page_elements / 8;
  const int at = piece * kCopyThreads * kCopyUnroll + threadIdx.x;
  uint4 x[kCopyUnroll];
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    if (at + i * kCopyThreads < chunks) x[i] = __ldcs(src + at + i * kCopyThreads);
  }
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    if (at + i * kCopyThreads < chunks) __stcs(dst + at + i * kCopyThreads, x[i]);
  }
}

// Compaction of the accepted drafted tokens: a block for one sequence, one layer, and K or V; a thread owns some 16-byte
// columns of the rows and carries every accepted token's column to its new place, eight at a time.  Places ascend and none
// lies behind its source, so a column that was read has been read before it is overwritten, whatever else the block does.
constexpr int kAcceptBatch = 8, kAcceptTile = 64;

__global__ void __launch_bounds__(256) accept_kernel(const AcceptParams p) {
  __shared__ long long from[kAcceptTile], to[kAcceptTile];
  const int b = blockIdx.x;
  const int drafted = p.drafted_offsets[b + 1] - p.drafted_offsets[b];
  const int base = p.lengths[b] - drafted;
  const int begin = p.accepted_offsets[b], count = p.accepted_offsets[b + 1] - begin;
  if (blockIdx.y == 0 && threadIdx.x == 0) p.new_lengths[b] = base + max(count, 0);
  uint16_t* cache = (blockIdx.y & 1 ? p.v : p.k) + (blockIdx.y >> 1) * p.layer_stride;
  const int row_chunks = p.head_dim / 8, columns = p.kv_heads * row_chunks;
  for (int tile = 0; tile < count; tile += kAcceptTile) {
    const int here = min(kAcceptTile, count - tile);
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * here; i += blockDim.x) {
      const int at = tile + i / 2;
      const int node = i & 1 ? at : p.accepted[begin + at];
      const int place = base + node;
      long long offset = -1;
      if (node >= 0 && node < drafted && place >= 0 && place / p.page_size < p.table_pages) {
        const int page = p.page_table[static_cast<long long>(b) * p.table_stride + place / p.page_size];
        if (page >= 0 && page < p.pages) offset = page * p.page_stride + (place % p.page_size) * p.token_stride;
      }
      (i & 1 ? to : from)[i / 2] = offset;
    }
    __syncthreads();
    for (int column = threadIdx.x; column < columns; column += blockDim.x) {
      const int head = column / row_chunks;
      uint16_t* mine = cache + head * p.head_stride + (column - head * row_chunks) * 8;
      for (int i0 = 0; i0 < here; i0 += kAcceptBatch) {
        uint4 x[kAcceptBatch];
#pragma unroll
        for (int i = 0; i < kAcceptBatch; ++i) {
          if (i0 + i < here && from[i0 + i] >= 0) x[i] = *reinterpret_cast<const uint4*>(mine + from[i0 + i]);
        }
#pragma unroll
        for (int i = 0; i < kAcceptBatch; ++i) {
          if (i0 + i < here && from[i0 + i] >= 0 && to[i0 + i] >= 0 && from[i0 + i] != to[i0 + i]) {
            *reinterpret_cast<uint4*>(mine + to[i0 + i]) = x[i];
          }
        }
      }
    }
  }
}

}  // namespace

template <int kThreads>
static cudaError_t launch_rotary_threads(const RotaryParams& p, int dtype, int tokens, cudaStream_t stream) {
  const int rows = p.q_heads + p.k_heads + p.v_heads;
  const dim3 block(p.head_dim / 16, kThreads / (p.head_dim / 16));
  const int tokens_per_block = std::min(16, std::max(tokens, static_cast<int>(block.y) / rows));
  const int grid = (p.tokens + tokens_per_block - 1) / tokens_per_block;
  const size_t smem = static_cast<size_t>(tokens_per_block) * (p.rotary_dim / 2) * sizeof(float2);
  if (dtype == FT_SRC_BF16) {
    rotary_kernel<__nv_bfloat162, kThreads><<<grid, block, smem, stream>>>(p, tokens_per_block);
  } else {
    rotary_kernel<__half2, kThreads><<<grid, block, smem, stream>>>(p, tokens_per_block);
  }
  return cudaGetLastError();
}

cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream) {
  if (p.tokens <= 0 || p.q_heads + p.k_heads + p.v_heads <= 0) return cudaSuccess;
  // Few tokens: a block of many threads per token, so that its rows go in one or two rounds (64 tokens: 2.4 us with 512 threads, 3.0
  // with 256).  Many: smaller blocks, of two tokens once that fills the SMs (16384 tokens: 64 us, 72 with 512 threads), or of
  // three where a block's last round is then fuller (5001 tokens of 16 + 4 heads, 40 or 60 rows in two rounds of 32: 13.6 and
  // 11.8 us; 16384 tokens of 32 + 8 + 8 heads, 96 rows in three rounds or 144 in five: 66.9 and 68.0).
  if (p.tokens <= 512) return launch_rotary_threads<512>(p, dtype, 1, stream);
  const int rows = p.q_heads + p.k_heads + p.v_heads, at_once = 256 / (p.head_dim / 16);
  const int rounds_of_two = (2 * rows + at_once - 1) / at_once, rounds_of_three = (3 * rows + at_once - 1) / at_once;
  const int tokens = p.tokens < 4096 ? 1 : 2 * rounds_of_three < 3 * rounds_of_two ? 3 : 2;
  return launch_rotary_threads<256>(p, dtype, tokens, stream);
}

static int pieces_of(int page_elements) { return (page_elements / 8 + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll); }

int copy_pages_most(int page_elements) { return 0x7fffffff / pieces_of(page_elements); }

cudaError_t launch_copy_pages(const CopyPagesParams& p, cudaStream_t stream) {
  if (p.count <= 0) return cudaSuccess;
  const int pieces = pieces_of(p.page_elements);
  copy_pages_kernel<<<dim3(static_cast<unsigned>(p.count) * pieces, 2 * p.layers), kCopyThreads, 0, stream>>>(p, pieces);
  return cudaGetLastError();
}

cudaError_t launch_accept(const AcceptParams& p, cudaStream_t stream) {
  if (p.batch <= 0) return cudaSuccess;
  const int columns = p.kv_heads * p.head_dim / 8;
  const int threads = std::min(256, (columns + 31) / 32 * 32);
  accept_kernel<<<dim3(p.batch, 2 * p.layers), threads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace ftg
