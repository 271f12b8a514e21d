// Attention of each sequence's queries over its keys, packed one behind the other or in the pages of a cache:
//   o_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = exp(scale q_t k_j) over the keys j that token t sees.
//
// One persistent CTA per SM takes an equal share of the 128-key tiles of the whole call (serving_schedule.h), so the
// lengths of the sequences do not matter to the balance, and a long context is split over as many CTAs as there are when
// there are few rows.  The query heads of a key head are rows of one tile (row = token * group + head in group), which
// reads K and V once for the group.  Two sides A and B work in turn, each on scores and an accumulator of its own:
//   kSplitKeys = false   two row tiles of 128 rows that share every K and V tile   (many rows)
//   kSplitKeys = true    one row tile; the sides take the even and the odd key tiles and merge at the end   (few rows)
// While one side is in its softmax the tensor core works for the other: scores S = Q K^T into tensor memory, the
// probabilities go back to tensor memory in 16 bits over the scores they came from, and are the left operand of
// O += P V.  A side has two warpgroups, one for each half of the 128 keys, so two threads share a row: one row per thread
// leaves a scheduler with a single warp per side, whose latencies nothing hides (4 x 4096 tokens, 32 heads of 128: 570 us
// against 498 us).  The exponent's reference follows the running maximum in steps of 2^8 only, so that the accumulator
// in tensor memory is hardly ever rescaled; the two threads of a row exchange their maxima through shared memory.
//
//   warp 0      walks the share: item descriptors for the others, tensor copies of Q, K and V
//   warp 1      one thread issues the matrix instructions
//   warp 2      clears what lies behind the last key in the tile of V that holds it
//   warps 3-6, 7-10, 11-14, 15-18   softmax of (A, first keys), (A, second), (B, first), (B, second); they write the output too
//
// A share that begins or ends inside a row tile leaves its part (unnormalised O, reference and sum of each row) in the
// workspace; serve_attention_combine_kernel adds the parts up.  Nothing depends on the order in which CTAs run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "serving_kernels.h"
#include "serving_schedule.h"
#include "sm100_ptx.cuh"

namespace ftg {

namespace {

constexpr int kRows = 128;     // rows of a tile: the lanes of tensor memory
constexpr int kRoleWarps = 3;  // in front of the softmax warps
// 96 registers each.  Nothing spills: spills would go to an L1 cache that shared memory has left little of.
constexpr int kThreads = (kRoleWarps + 16) * 32;
// A role that has nothing to do for an item waits while the others go through its keys: up to 2^20 tiles of them (2^27 keys), at
// 2.1 us for two tiles of rows with heads of 128 and 1.9 GHz, 3.1 where the power cap holds the clock at 1.3 GHz.  (The timer's
// low word counts to 4.29 s.)
constexpr uint32_t kTimeoutNs = 4000000000u;
constexpr float kRescaleStep = 8.0f;  // log2 units
constexpr int kItems = 4;             // descriptors in flight
// The tensor core cuts each product off some 2^-25 below the sum it is added to, always towards zero: over N keys that is up to
// N 2^-27 of the sum (equal values, one row tile per CTA: 0.5 % too small after 2^20 keys, 11 % after 2^24).  After so many of its
// key tiles a side adds its accumulator to a copy in the workspace and begins anew, so no more than 2^17 keys, 2^-10, weigh on a sum.
constexpr int kKeepTiles = 1024;
constexpr int kMaxStages = 12;
constexpr uint32_t kTmemS = 0, kTmemO = 256;  // S of A and B: 128 columns each; O of A and B: kDim each

struct Item {
  int token0;      // first query row in q and out
  int tokens;      // queries of this row tile; negative: the walk is over
  int place0;      // place of the first query among the sequence's queries
  int kv_head;
  int prefix, keys, limit;  // limit: no row sees a key at or behind it
  int first, end;  // key tiles of this part
  int slot;        // -1: the whole row tile, straight to the output; otherwise which part in the workspace
};

struct Shared {
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_full[2], o_full[2], o_empty[2];
  uint64_t tail_wanted, tail_cleared;
  uint64_t item_full[kItems], item_empty[kItems];
  Item items[kItems];
  uint32_t tmem_base;
  int abort_flag;
  uint64_t max_ready[2][4];  // [side][quarter]: both warps of the rows have written the maxima of their keys
  uint64_t state_full[2];    // [side] (kSplitKeys: the first for both)
  float row_max[2][2][kRows];     // [side][key half]; written again only when the next scores are there, which follows both reads
  float2 state[2][2][2][kRows];   // [item parity][side][key half]: {reference, sum} of the rows, in turn for odd and even items
  float2 kept[2][2][kRows];       // [side][key half]: {reference, sum} of what the sides have put into the workspace
};

template <int kDim, bool kSplitKeys>
struct Layout {
  static constexpr int kSlabs = kDim / 64;              // 128-byte columns of a row of Q, K or V
  static constexpr int kTileBytes = kSlabs * 128 * 128;
  static constexpr int kQTiles = kSplitKeys ? 1 : 2;
  // What a row tile costs beside its key tiles, in key tiles.  Split, 64 single tokens over up to 8060 keys take 89, 69, 75
  // and 79 us at 1, 2, 3 and 4; in pairs, twenty ragged prompts with heads of 64 take 180, 190 and 202 at 1, 2 and 3, with
  // heads of 128 and on fewer heads 123, 121 and 128.
  static constexpr int kItemCost = kSplitKeys || kDim == 128 ? 2 : 1;
  static constexpr int kStages = kDim == 64 ? 10 : kSplitKeys ? 5 : 4;
  static constexpr int kBytes = (kQTiles + kStages) * kTileBytes + static_cast<int>(sizeof(Shared)) + 1024;
  static_assert(kBytes <= 232448 && kStages <= kMaxStages, "shared memory of one CTA");
};

// The workspace: what a combining block has to know per CTA, then {reference, sum} and O of the parts, [slot][half][..].
struct Unfinished {
  int valid, last_cta;  // the row tile that begins in this CTA and ends in last_cta
  int token0, tokens, kv_head, pad;
};
struct Parts {
  Unfinished* unfinished;  // [cta]
  float2* state;           // [cta][2 slots][2 halves][128]
  float4* o;               // [cta][2][2][kDim / 4][128]
};
__host__ __device__ inline Parts parts_of(void* workspace, int ctas) {
  Parts parts;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  parts.unfinished = reinterpret_cast<Unfinished*>(at);
  at += (static_cast<size_t>(ctas) * sizeof(Unfinished) + 255) / 256 * 256;
  parts.state = reinterpret_cast<float2*>(at);
  at += static_cast<size_t>(ctas) * 4 * kRows * sizeof(float2);
  parts.o = reinterpret_cast<float4*>(at);
  return parts;
}
size_t parts_bytes(int ctas) {
  return (static_cast<size_t>(ctas) * sizeof(Unfinished) + 255) / 256 * 256 + static_cast<size_t>(ctas) * 4 * kRows * (sizeof(float2) + 128 * sizeof(float));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The same on the FMA pipe: x = r + f with r a whole number (adding 1.5 * 2^23 rounds to it) and |f| <= 1/2; 2^f is the
// polynomial of degree 5 with the smallest relative error there and a constant term of 1 (fitted by least squares, reweighted
// towards the largest errors; with these constants 1.1e-7 in exact arithmetic, 1.7e-7 in 32 bits), 2^r goes into the exponent bits.  At -127 and below the
// result is 0, and a NaN stays one.
__device__ __forceinline__ float exp2_polynomial(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(y) : "f"(x));
  const float t = y + 12582912.0f;
  const float f = y - (t - 12582912.0f);
  float p = fmaf(0.00132647273f, f, 0.00967151299f);
  p = fmaf(p, f, 0.0555073358f);
  p = fmaf(p, f, 0.240222424f);
  p = fmaf(p, f, 0.693147004f);
  p = fmaf(p, f, 1.0f);
  return p * __int_as_float((__float_as_int(t) << 23) + (127 << 23));
}
// Two numbers to 16 bits, the first in the low half.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (kBf16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

// The smallest normal fp16 is 2^-14: the probabilities are carried times 2^7 there (at most 2^15 with the lagging
// reference), so that keys far below the maximum keep their precision.  bf16 has the range of FP32.
template <bool kBf16>
constexpr float kShift = kBf16 ? 0.0f : 7.0f;

// mbar_wait_bounded in few instructions (it stands in some thirty places): gives up after kTimeoutNs, or when another role has.
__device__ __forceinline__ uint32_t timer_lo() {
  uint32_t t;
  asm volatile("mov.u32 %0, %globaltimer_lo;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t start = timer_lo();
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag != 0 || timer_lo() - start > kTimeoutNs) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffU, wait_for(bar, parity, abort_flag));
}

__device__ __forceinline__ void tma_load_3d(void* smem, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* smem, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* smem, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w, int u) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(smem)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u)
               : "memory");
}
// Shared-memory matrix descriptors (128-byte swizzle, 8 rows of 128 bytes per 1024): the high word is a constant, the low
// word holds the start address / 16 and, in bits 16 and up, the leading byte offset / 16.  Only the low word is kept in
// registers: as 64-bit values the descriptors of an unrolled tile take more than a thread has.
// group_stride: bytes from 8 rows to the next 8
__host__ __device__ constexpr uint32_t desc_high(uint32_t group_stride) { return (group_stride >> 4) | (1u << 14) | (2u << 29); }
constexpr uint32_t kDescRows = 1u << 16;                    // K-major (Q, K); the offset is not used

// Where a tile of K or V has its rows: 8 rows of 128 bytes (64 elements, a slab) lie together.  Packed prompts: slab by slab,
// 128 rows each.  Pages: the slabs of 8 rows side by side, so that one copy brings all slabs of a page: with one copy for each,
// 64 single tokens over 262000 keys in all (heads of 128) took 246 us against 196 in pages of 16, 371 against 248 in pages of 8,
// 188 against 175 in pages of 32 (173 in larger ones).
struct TileRows {
  uint32_t group, slab;  // bytes from 8 rows to the next 8, from a slab to the next
  __device__ __forceinline__ TileRows(int slabs, bool paged) : group(paged ? slabs * 1024 : 1024), slab(paged ? 1024 : 128 * 128) {}
};

// D[tmem] (+)= A[smem] * B[smem]^T, 16-bit operands.
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t b_high, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %6};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(b_high), "n"(desc_high(1024))
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]; A holds two elements per column.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t b_high, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b), "r"(idesc), "r"(accumulate), "r"(b_high)
      : "memory");
}
// Instruction descriptor of kind::f16: FP32 accumulator, both operands bf16 (1) or fp16 (0); bit 16: B is N-major.
template <bool kBf16>
__host__ __device__ constexpr uint32_t idesc16(int n, bool b_n_major) {
  return (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (b_n_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
// What the call's arrays say about sequence b, cut to what may be read.
struct Sequence {
  int token0, key_row0;
  SequenceTiles tiles;
};
struct RawSequence {
  int q_begin, q_end, k_begin, k_end;
};
__device__ __forceinline__ RawSequence load_raw(const ServeAttentionParams& p, int b) {
  RawSequence r;
  r.q_begin = p.q_offsets[b];
  r.q_end = p.q_offsets[b + 1];
  r.k_begin = p.page_table != nullptr ? 0 : p.k_offsets[b];
  r.k_end = p.page_table != nullptr ? p.lengths[b] : p.k_offsets[b + 1];
  return r;
}
__device__ __forceinline__ Sequence make_sequence(const ServeAttentionParams& p, const RawSequence& r, int tokens_per_item, int item_cost) {
  Sequence s;
  s.token0 = min(max(r.q_begin, 0), p.query_tokens);
  const int queries = min(max(r.q_end, s.token0), p.query_tokens) - s.token0;
  int keys, full;
  if (p.page_table != nullptr) {
    s.key_row0 = 0;
    full = max(r.k_end, 0);
    keys = min(full, p.table_pages * p.page_size);
  } else {
    s.key_row0 = min(max(r.k_begin, 0), p.key_tokens);
    keys = full = min(max(r.k_end, s.key_row0), p.key_tokens) - s.key_row0;
  }
  s.tiles = SequenceTiles::make(queries, keys, full, tokens_per_item, item_cost, p.causal != 0 && p.mask == nullptr);
  return s;
}

__device__ __forceinline__ Sequence load_sequence(const ServeAttentionParams& p, int b, int tokens_per_item, int item_cost) {
  return make_sequence(p, load_raw(p, b), tokens_per_item, item_cost);
}

__device__ __forceinline__ Item load_item(const volatile Item& from) {
  Item i;
  i.token0 = from.token0;
  i.tokens = from.tokens;
  i.place0 = from.place0;
  i.kv_head = from.kv_head;
  i.prefix = from.prefix;
  i.keys = from.keys;
  i.limit = from.limit;
  i.first = from.first;
  i.end = from.end;
  i.slot = from.slot;
  return i;
}

// Where a warpgroup keeps its half of the columns of its side's accumulator, [column / 4][row]: the place of the item's own part, or,
// for a whole row tile, of the part that only the CTA's last item can have.
template <int kDim>
__device__ __forceinline__ float4* kept_at(void* workspace, int slot, int side, int column_half) {
  return parts_of(workspace, gridDim.x).o + (((static_cast<size_t>(blockIdx.x) * 2 + (slot < 0 ? 1 : slot)) * 2 + side) * (kDim / 4) + column_half * (kDim / 8)) * kRows;
}
// Adds this thread's columns of the accumulator and its sum to what is kept (`again`: something is) and begins anew; or, `back`,
// adds what is kept to the accumulator and to the sum that it returns.
template <int kDim>
__device__ __forceinline__ float keep_accumulator(uint32_t o_addr, float4* o_kept, float2* kept, float reference, float sum, bool again, bool back) {
  tcgen05_fence_after();
  float shrink = 0.0f;
  if (again) {
    shrink = exp2_approx(kept->x - (reference == -INFINITY ? 0.0f : reference));
    sum = fmaf(kept->y, shrink, sum);
  }
#pragma unroll 1
  for (int d = 0; d < kDim / 2; d += 8, o_kept += 2 * kRows) {
    float o[8];
    tmem_ld_32x32b_x8(o_addr + d, o);
    tmem_wait_ld();
    if (again) {
      const float4 a = o_kept[0], b = o_kept[kRows];
      o[0] = fmaf(a.x, shrink, o[0]);
      o[1] = fmaf(a.y, shrink, o[1]);
      o[2] = fmaf(a.z, shrink, o[2]);
      o[3] = fmaf(a.w, shrink, o[3]);
      o[4] = fmaf(b.x, shrink, o[4]);
      o[5] = fmaf(b.y, shrink, o[5]);
      o[6] = fmaf(b.z, shrink, o[6]);
      o[7] = fmaf(b.w, shrink, o[7]);
    }
    if (!back) {
      o_kept[0] = make_float4(o[0], o[1], o[2], o[3]);
      o_kept[kRows] = make_float4(o[4], o[5], o[6], o[7]);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = 0.0f;
    }
    tmem_st_32x32b_x8(o_addr + d, o);
  }
  tmem_wait_st();
  tcgen05_fence_before();
  if (back) return sum;
  *kept = make_float2(reference, sum);
  return 0.0f;
}

template <int kDim>
__device__ __noinline__ float keep_accumulator_call(uint32_t o_addr, float4* o_kept, float2* kept, float reference, float sum, bool again) {
  return keep_accumulator<kDim>(o_addr, o_kept, kept, reference, sum, again, false);
}

// In pairs the unit for exponentials has as much to do as the tensor core (a tile's 128 x 128 take it 1024 cycles, the two
// products with heads of 128 as many), so one exponential in eight goes to the FMA pipe: the pairs of numbers e of the
// sixteen of a half.  B200, 4 x 4096 tokens, 32 heads, us without and with: heads of 64 849 -> 712 (causal 466 -> 390), heads of
// 128 causal 508 -> 498.  Three pairs of sixteen: 815 and 525; one: 760 and 505; other places for two: 726 to 790 and 500 to 520.
// One row tile waits for other things more: trees over up to 7700 keys 71.4 -> 72.7.
template <int kDim, bool kSplitKeys>
__device__ constexpr bool by_polynomial(int e) {
  return !kSplitKeys && (e == 11 || e == (kDim == 64 ? 3 : 15));
}

// The queries of side `half` and the key tiles it works through.
template <bool kSplitKeys>
struct HalfWork {
  int place0, tokens;  // its first query's place among the item's, how many
  int count;           // key tiles
  __device__ __forceinline__ HalfWork(const Item& item, int half, int tokens_per_half, bool chain) {
    const int n = item.end - item.first;
    if (kSplitKeys) {
      place0 = 0;
      tokens = item.tokens;
      count = (n + 1 - half) / 2;
    } else {
      place0 = half * tokens_per_half;
      tokens = min(max(item.tokens - place0, 0), tokens_per_half);
      const int limit = tokens == 0 ? 0 : chain ? min(item.limit, item.prefix + item.place0 + place0 + tokens) : item.limit;
      const int tiles = limit <= 0 ? 0 : (limit - 1) / kKeyTile + 1;
      count = min(max(tiles - item.first, 0), n);
    }
  }
};

}  // namespace

template <int kDim, bool kBf16, bool kSplitKeys, bool kPaged>
__global__ void __launch_bounds__(kThreads, 1)
serve_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                       const __grid_constant__ ServeAttentionParams p) {
  using L = Layout<kDim, kSplitKeys>;
  extern __shared__ uint8_t smem_raw[];
  // aligned by arithmetic on the shared array itself, which keeps the accesses in the shared address space
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* smem_q = smem;
  uint8_t* smem_kv = smem + L::kQTiles * L::kTileBytes;
  Shared& sh = *reinterpret_cast<Shared*>(smem_kv + L::kStages * L::kTileBytes);
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = __shfl_sync(0xffffffffU, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // warp: in a uniform register
  const int tokens_per_half = p.tokens_per_tile;
  const int tokens_per_item = L::kQTiles * tokens_per_half;
  const bool chain = p.causal != 0 && !(kPaged && p.mask != nullptr);

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.tail_wanted, 1);
    mbar_init(&sh.tail_cleared, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 8);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], kSplitKeys ? 16 : 8);
      mbar_init(&sh.state_full[i], kSplitKeys ? 16 : 8);
      for (int quarter = 0; quarter < 4; ++quarter) mbar_init(&sh.max_ready[i][quarter], 2);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_empty[i], 18);
    }
    sh.abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmap_q);
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  // Everything above may run while the kernel in front on the stream still does; nothing below may.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's share (warp 0): the lanes sum up the sequences' units, a stretch of sequences each
  Sequence seq = {};
  int first_sequence = 0;
  int left = 0, start = 0, share = 0, per_head = 1;  // units of the share; in front of it in its sequence; per CTA; per key head
  if (warp == 0) {
    int batch = p.batch;
    if (p.count_units != 0) {
      long long most = 0;
#pragma unroll 1
      for (int i = lane; i < p.batch; i += 32) most += load_sequence(p, i, tokens_per_item, L::kItemCost).tiles.most_units_per_head() * p.kv_heads;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) most += __shfl_xor_sync(0xffffffffU, most, off);
      if (most > 0x7fffffff) {  // nothing is done
        batch = 0;
        if (blockIdx.x == 0 && lane == 0) atomicExch(p.status, FT_ERR_INVALID);
      }
    }
    const int per_lane = (batch + 31) / 32;
    const int scan_begin = min(lane * per_lane, batch), scan_end = min(scan_begin + per_lane, batch);
    int mine = 0, before = 0, share_begin = 0, at = 0, found = scan_begin;
    bool holds = false;
    // first the sums; then the lane whose stretch holds the beginning goes through it once more, unless it is one sequence
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
      for (int i = scan_begin; i < scan_end; ++i) {
        seq = load_sequence(p, i, tokens_per_item, L::kItemCost);
        per_head = seq.tiles.units_per_head();
        const int units = per_head * p.kv_heads;
        if (pass == 0) {
          mine += units;
        } else {
          found = i;
          if (share_begin < at + units) break;
          at += units;
        }
      }
      if (pass == 1) break;
      before = mine;  // inclusive prefix
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int other = __shfl_up_sync(0xffffffffU, before, off);
        if (lane >= off) before += other;
      }
      const int total = __shfl_sync(0xffffffffU, before, 31);
      before -= mine;
      share = total / static_cast<int>(gridDim.x) + 1;
      share_begin = static_cast<int>(min(static_cast<long long>(share) * blockIdx.x, static_cast<long long>(total)));
      left = min(share, total - share_begin);
      holds = left > 0 && before <= share_begin && share_begin < before + mine;
      at = before;
      if (!holds || per_lane == 1) break;
    }
    __syncwarp();
    const unsigned holders = __ballot_sync(0xffffffffU, holds);
    if (holders == 0) left = 0;
    if (left > 0) {
      const int owner = __ffs(holders) - 1;
      first_sequence = __shfl_sync(0xffffffffU, found, owner);
      start = share_begin - __shfl_sync(0xffffffffU, at, owner);
      per_head = __shfl_sync(0xffffffffU, per_head, owner);
      seq.token0 = __shfl_sync(0xffffffffU, seq.token0, owner);
      seq.key_row0 = __shfl_sync(0xffffffffU, seq.key_row0, owner);
      seq.tiles.queries = __shfl_sync(0xffffffffU, seq.tiles.queries, owner);
      seq.tiles.keys = __shfl_sync(0xffffffffU, seq.tiles.keys, owner);
      seq.tiles.prefix = __shfl_sync(0xffffffffU, seq.tiles.prefix, owner);
      seq.tiles.row_tiles = __shfl_sync(0xffffffffU, seq.tiles.row_tiles, owner);
      seq.tiles.tokens_per_item = tokens_per_item;
      seq.tiles.item_cost = L::kItemCost;
      seq.tiles.chain = chain;
      seq.tiles.ramp = __shfl_sync(0xffffffffU, seq.tiles.ramp ? 1 : 0, owner) != 0;
      // offsets that do not ascend can promise more than 31 bits of work: a share outside its sequence is left out
      if (start < 0 || start / p.kv_heads >= per_head) left = 0;
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = sh.tmem_base;

  if (warp < kRoleWarps) {
    if (warp == 0) {
      // ------------------------------------------------------------- the walk, and the tensor copies
      int b = first_sequence;
      Unfinished unfinished = {};
      int stage = 0, stage_phase = 0, q_phase = 0;
      uint32_t item_index = 0;
      bool ok = true;
      int kv_head = 0, row_tile = 0, first = 0;
      if (left > 0) {
        kv_head = start / per_head;
        const int inner = start - kv_head * per_head;
        int lo = 0, in_front = 0;  // units_before(lo) <= inner
        if (seq.tiles.ramp) {
#pragma unroll 1
          for (int hi = seq.tiles.row_tiles; hi - lo > 1;) {
            const int step = (hi - lo + 31) / 32;
            const int probe = min(lo + lane * step, hi);
            const int units = seq.tiles.units_before(probe);
            const int last = __popc(__ballot_sync(0xffffffffU, probe < hi && units <= inner)) - 1;
            in_front = __shfl_sync(0xffffffffU, units, last);
            lo = lo + last * step;
            hi = min(lo + step, hi);
          }
        } else {
          lo = inner / seq.tiles.units_of(0);
          in_front = lo * seq.tiles.units_of(0);
        }
        row_tile = lo;
        first = inner - in_front;
        if (first <= L::kItemCost) {  // the whole row tile is this CTA's, whatever lies in front of the boundary
          left += first;
          first = 0;
        }
      }
      RawSequence next = load_raw(p, min(b + 1, p.batch - 1));  // a sequence ahead
      while (ok) {
        const int slot_index = item_index % kItems;
        ok = warp_wait(&sh.item_empty[slot_index], ((item_index / kItems) & 1) ^ 1, abort_flag);
        if (!ok) break;
        Item item = {};
        const int units = left > 0 ? seq.tiles.units_of(row_tile) : 0;
        if (left <= 0 || (first == 0 && left <= L::kItemCost && left < units)) {  // the next CTA takes a row tile that would only begin here
          item.tokens = -1;
          if (lane == 0) {
            sh.items[slot_index] = item;
            mbar_arrive(&sh.item_full[slot_index]);
          }
          break;
        }
        const int end = min(units, first + left);
        item.place0 = row_tile * tokens_per_item;
        item.token0 = seq.token0 + item.place0;
        item.tokens = min(seq.tiles.queries - item.place0, tokens_per_item);
        item.kv_head = kv_head;
        item.prefix = seq.tiles.prefix;
        item.keys = seq.tiles.keys;
        item.limit = seq.tiles.limit(item.place0 + item.tokens);
        const int real = item.limit <= 0 ? 0 : (item.limit - 1) / kKeyTile + 1;  // a unit may have no key tile in it
        item.first = min(max(first - L::kItemCost, 0), real);
        item.end = min(max(end - L::kItemCost, 0), real);
        item.slot = first == 0 && end == units ? -1 : first > 0 ? 0 : 1;
        if (first == 0 && end < units) {
          unfinished.valid = 1;
          unfinished.last_cta = min(static_cast<int>(blockIdx.x) + (units - end + share - 1) / share, static_cast<int>(gridDim.x) - 1);
          unfinished.token0 = item.token0;
          unfinished.tokens = item.tokens;
          unfinished.kv_head = kv_head;
        }
        if (lane == 0) {
          sh.items[slot_index] = item;
          mbar_arrive(&sh.item_full[slot_index]);
        }
        ++item_index;

        // tensor copies of this part: lane 0 alone, or a lane for each page
        const int tiles = item.end - item.first;
        if (tiles > 0) {
          ok = warp_wait(&sh.q_empty, q_phase ^ 1, abort_flag);
          if (!ok) break;
          q_phase ^= 1;
          const int q_tiles = kSplitKeys || item.tokens <= tokens_per_half ? 1 : 2;
          if (lane == 0) {
            mbar_arrive_expect_tx(&sh.q_full, q_tiles * L::kSlabs * tokens_per_half * p.group * 128);
            for (int t = 0; t < q_tiles; ++t) {
#pragma unroll
              for (int sl = 0; sl < L::kSlabs; ++sl) {
                tma_load_4d(smem_q + t * L::kTileBytes + sl * (128 * 128), &tmap_q, &sh.q_full, 64 * sl, 0, kv_head, item.token0 + t * tokens_per_half);
              }
            }
          }
          const int box = min(p.page_size, kKeyTile);
          // lane i holds the page of the i-th box of a key tile, asked for a tile ahead; behind the limit nothing is read
          auto boxes_of = [&](int tile) { return (min(item.limit - tile * kKeyTile, kKeyTile) + box - 1) / box; };
          auto page_of = [&](int tile) -> int {
            int page = 0;
            if (kPaged && tile < item.end && lane < boxes_of(tile)) {
              page = p.page_table[static_cast<long long>(b) * p.table_stride + (tile * kKeyTile + lane * box) / p.page_size];
            }
            return page;
          };
          auto load = [&](const CUtensorMap* map, int tile, int page) -> bool {
            if (!warp_wait(&sh.kv_empty[stage], stage_phase ^ 1, abort_flag)) return false;
            uint8_t* to = smem_kv + stage * L::kTileBytes;
            if (!kPaged) {
              if (lane == 0) {
                mbar_arrive_expect_tx(&sh.kv_full[stage], L::kTileBytes);
#pragma unroll
                for (int sl = 0; sl < L::kSlabs; ++sl) {
                  tma_load_3d(to + sl * (128 * 128), map, &sh.kv_full[stage], 64 * sl, kv_head, seq.key_row0 + tile * kKeyTile);
                }
              }
            } else {
              const int boxes = boxes_of(tile);
              if (lane == 0) mbar_arrive_expect_tx(&sh.kv_full[stage], boxes * box * L::kSlabs * 128);
              __syncwarp();
              if (lane < boxes) {
                const int place = (tile * kKeyTile + lane * box) & (p.page_size - 1);
                const bool known = page >= 0 && page < p.pages;  // otherwise outside the tensor: filled with zeros
                tma_load_5d(to + lane * box * (L::kSlabs * 128), map, &sh.kv_full[stage], 0, 0, 0, (known ? page : p.pages) * p.page_groups + place / 8, kv_head);
              }
            }
            if (++stage == L::kStages) {
              stage = 0;
              stage_phase ^= 1;
            }
            return true;
          };
          int page_v = page_of(item.first), page_k = page_of(item.first + 1), page_ahead = page_of(item.first + 2);
          ok = load(&tmap_k, item.first, page_v);
          for (int t = item.first; ok && t < item.end; ++t) {
            if (kSplitKeys) {
              if (t + 1 < item.end) ok = load(&tmap_k, t + 1, page_k);
              if (ok) ok = load(&tmap_v, t, page_v);
            } else {
              ok = load(&tmap_v, t, page_v);
              if (ok && t + 1 < item.end) ok = load(&tmap_k, t + 1, page_k);
            }
            page_v = page_k;
            page_k = page_ahead;
            page_ahead = page_of(t + 3);
          }
        }
        // the next part
        left -= end - first;
        first = 0;
        if (left > 0 && ++row_tile == seq.tiles.row_tiles) {
          row_tile = 0;
          if (++kv_head == p.kv_heads) {
            kv_head = 0;
            do {
              ++b;
              seq = make_sequence(p, next, tokens_per_item, L::kItemCost);
              next = load_raw(p, min(b + 1, p.batch - 1));
            } while (seq.tiles.row_tiles == 0 && b + 1 < p.batch);
            // offsets that do not ascend may promise more than there is: nothing is read behind the last sequence
            if (b >= p.batch || seq.tiles.row_tiles == 0) left = 0;
          }
        }
      }
      if (lane == 0) parts_of(p.workspace, gridDim.x).unfinished[blockIdx.x] = unfinished;
      // every stage is empty again before the CTA leaves: nothing arrives on its barriers any more
      for (int i = 0; ok && i < L::kStages; ++i) {
        ok = warp_wait(&sh.kv_empty[stage], stage_phase ^ 1, abort_flag);
        if (++stage == L::kStages) {
          stage = 0;
          stage_phase ^= 1;
        }
      }
      if (ok) warp_wait(&sh.q_empty, q_phase ^ 1, abort_flag);
    } else if (warp == 1) {
      // ------------------------------------------------------------- matrix instructions, all by one thread
      if (elect_one()) {
        constexpr uint32_t kIdescS = idesc16<kBf16>(128, false), kIdescO = idesc16<kBf16>(kDim, true);
        int stage = 0, stage_phase = 0, q_phase = 0, tail_phase = 0;
        uint32_t p_phase[2] = {0, 0}, o_phase[2] = {0, 0};
        bool ok = true;
        const uint32_t q_desc = (smem_u32(smem_q) >> 4) | kDescRows;
        const TileRows rows(L::kSlabs, kPaged);
        const uint32_t kv_high = desc_high(rows.group);
        const uint32_t k_desc = (smem_u32(smem_kv) >> 4) | kDescRows, v_desc = (smem_u32(smem_kv) >> 4) | (rows.slab >> 4 << 16);  // V: along N, slab by slab
        auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(bar, parity, abort_flag); };

        auto issue_s = [&](int x, int k_stage) {
          const uint32_t a = q_desc + (kSplitKeys ? 0 : x) * (L::kTileBytes >> 4), bd = k_desc + k_stage * (L::kTileBytes >> 4);
#pragma unroll
          for (int k = 0; k < kDim / 16; ++k) {
            umma_ss(tmem_base + kTmemS + x * 128, a + (k / 4) * ((128 * 128) >> 4) + (k % 4) * 2, bd + (k / 4) * (rows.slab >> 4) + (k % 4) * 2, kv_high,
                    kIdescS, k > 0);
          }
          umma_commit(&sh.s_full[x]);
        };
        auto next_stage = [&]() {
          if (++stage == L::kStages) {
            stage = 0;
            stage_phase ^= 1;
          }
        };

        for (uint32_t index = 0; ok; ++index) {
          const int slot_index = index % kItems;
          ok = wait(&sh.item_full[slot_index], (index / kItems) & 1);
          if (!ok) break;
          const Item item = sh.items[slot_index];
          mbar_arrive(&sh.item_empty[slot_index]);
          if (item.tokens < 0) break;
          const int n = item.end - item.first;
          if (n <= 0) continue;
          const int count[2] = {HalfWork<kSplitKeys>(item, 0, tokens_per_half, chain).count, HalfWork<kSplitKeys>(item, 1, tokens_per_half, chain).count};
          ok = wait(&sh.q_full, q_phase);
          if (!ok) break;
          q_phase ^= 1;

          // The tile of V in `v_stage` is there.  Behind the last key that anyone sees it holds whatever memory holds; the
          // probabilities there are zero, but zero times NaN is not, so the product stops at the next multiple of 16 keys and
          // warp 2 clears the rows up to it.
          auto steps_of = [&](int tile) -> int {
            const int valid = item.limit - tile * kKeyTile;
            if (valid >= kKeyTile) return 8;
            if (valid % 16 != 0) {
              mbar_arrive(&sh.tail_wanted);
              ok = wait(&sh.tail_cleared, tail_phase);
              tail_phase ^= 1;
            }
            return (valid + 15) / 16;
          };
          // O += P V of side x for the key tile in v_stage, its i-th; the probabilities of its first 64 keys lie where their
          // scores were, those of the others too.  Each product adds to all columns of O, and when the reference moves each
          // warpgroup rescales one half of them: even the products of the first 64 keys wait for both.  (B200, 4 x 4096
          // tokens: 496 to 505 us, and 502 where the two warps of a row meet behind a rescale instead; ragged prompts 44 to 45 and 45.4.)
          auto accumulate = [&](int x, int i, int v_stage, int steps) -> bool {
            if (i == 0) {
              if (!wait(&sh.o_empty[x], o_phase[x] ^ 1)) return false;
              o_phase[x] ^= 1;
            }
            const uint32_t bd = v_desc + v_stage * (L::kTileBytes >> 4);
            if (!wait(&sh.p_full[x], p_phase[x])) return false;
            tcgen05_fence_after();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if (k < steps) {
                umma_ts(tmem_base + kTmemO + x * kDim, tmem_base + kTmemS + x * 128 + (k / 4) * 64 + (k % 4) * 8, bd + k * (rows.group >> 3), kv_high, kIdescO,
                        i > 0 || k > 0);
              }
            }
            p_phase[x] ^= 1;
            if (i + 1 == count[x]) umma_commit(&sh.o_full[x]);
            return true;
          };

          if (kSplitKeys) {
            for (int t = 0; ok && t < min(n, 2); ++t) {
              ok = wait(&sh.kv_full[stage], stage_phase);
              if (!ok) break;
              tcgen05_fence_after();
              issue_s(t, stage);
              umma_commit(&sh.kv_empty[stage]);
              if (t + 1 == n) umma_commit(&sh.q_empty);
              next_stage();
            }
            for (int t = 0; ok && t < n; ++t) {
              const int x = t & 1;
              ok = wait(&sh.kv_full[stage], stage_phase);
              if (!ok) break;
              const int steps = steps_of(item.first + t);
              if (ok) ok = accumulate(x, t >> 1, stage, steps);
              if (!ok) break;
              umma_commit(&sh.kv_empty[stage]);
              next_stage();
              if (t + 2 < n) {
                ok = wait(&sh.kv_full[stage], stage_phase);
                if (!ok) break;
                tcgen05_fence_after();
                issue_s(x, stage);
                umma_commit(&sh.kv_empty[stage]);
                if (t + 3 == n) umma_commit(&sh.q_empty);
                next_stage();
              }
            }
          } else {
            ok = wait(&sh.kv_full[stage], stage_phase);
            if (!ok) break;
            tcgen05_fence_after();
            if (count[0] > 0) issue_s(0, stage);
            if (count[1] > 0) issue_s(1, stage);
            umma_commit(&sh.kv_empty[stage]);
            if (n == 1) umma_commit(&sh.q_empty);
            next_stage();
            for (int j = 0; ok && j < n; ++j) {
              const int v_stage = stage;
              ok = wait(&sh.kv_full[stage], stage_phase);
              if (!ok) break;
              next_stage();
              const int k_stage = stage;
              if (j + 1 < n) {
                ok = wait(&sh.kv_full[k_stage], stage_phase);
                if (!ok) break;
                next_stage();
              }
              const int steps = steps_of(item.first + j);
              for (int x = 0; ok && x < 2; ++x) {
                if (j >= count[x]) continue;
                ok = accumulate(x, j, v_stage, steps);
                if (ok && j + 1 < count[x]) issue_s(x, k_stage);
              }
              if (!ok) break;
              umma_commit(&sh.kv_empty[v_stage]);
              if (j + 1 < n) umma_commit(&sh.kv_empty[k_stage]);
              if (j + 2 == n) umma_commit(&sh.q_empty);
            }
          }
        }
      }
    } else {
      // ------------------------------------------------------------- rows of V behind the last key
      const TileRows rows(L::kSlabs, kPaged);
      int stage = 0, tail_phase = 0;
      for (uint32_t index = 0;; ++index) {
        const int slot_index = index % kItems;
        if (!warp_wait(&sh.item_full[slot_index], (index / kItems) & 1, abort_flag)) break;
        const Item item = sh.items[slot_index];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.item_empty[slot_index]);
        if (item.tokens < 0) break;
        const int n = item.end - item.first;
        if (n <= 0) continue;
        stage = (stage + 2 * n) % L::kStages;  // of the 2 n stages that this part goes through, the last holds the tile
        const int valid = item.limit - (item.end - 1) * kKeyTile;
        if (valid < kKeyTile && valid % 16 != 0) {
          if (!warp_wait(&sh.tail_wanted, tail_phase, abort_flag)) break;
          tail_phase ^= 1;
          uint8_t* v = smem_kv + (stage + L::kStages - 1) % L::kStages * L::kTileBytes;
          const int upto = (valid + 15) / 16 * 16;
          for (int i = lane; i < (upto - valid) * L::kSlabs * 8; i += 32) {
            const int row = valid + i / (L::kSlabs * 8), chunk = i % (L::kSlabs * 8);
            *reinterpret_cast<uint4*>(v + (chunk / 8) * rows.slab + (row / 8) * rows.group + (row % 8) * 128 + (chunk % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.tail_cleared);
        }
      }
    }
  } else {
    // --------------------------------------------------------------- softmax: two threads per row, 64 keys each
    const int group_index = (warp - kRoleWarps) >> 2;
    const int x = group_index >> 1, c = group_index & 1;  // side, key half
    const int quarter = warp & 3;                         // the lanes of tensor memory this warp can reach
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter) << 21;  // lane index in bits 16 and up, 32 lanes per warp
    const uint32_t s_addr = tmem_base + lanes + kTmemS + x * 128 + c * 64;
    const uint32_t o_addr = tmem_base + lanes + kTmemO + x * kDim + c * (kDim / 2);
    const int row_token = row / p.group;
    uint32_t s_phase = 0, o_phase = 0, max_phase = 0;
    bool ok = true;

    for (uint32_t index = 0; ok; ++index) {
      const int slot_index = index % kItems;
      ok = warp_wait(&sh.item_full[slot_index], (index / kItems) & 1, abort_flag);
      if (!ok) break;
      // The descriptor stays in shared memory until the row tile is done: the loop over its key tiles needs the registers
      // (what it spills goes to an L1 cache that shared memory has left next to nothing of).
      volatile Item& item = sh.items[slot_index];
      if (item.tokens < 0) break;
      int count, plain;  // key tiles of this side; every key below `plain` is seen, with a mask its bits say which of the rest are
      bool real_row;
      {
        const Item copy = load_item(item);
        const HalfWork<kSplitKeys> work(copy, x, tokens_per_half, chain);
        count = work.count;
        real_row = row_token < min(work.tokens, tokens_per_half);
        plain = !real_row          ? 0
                : (kPaged && p.mask != nullptr) ? min(copy.prefix, copy.keys)
                : chain             ? min(copy.limit, copy.prefix + copy.place0 + work.place0 + row_token + 1)
                                    : copy.keys;
      }
      const bool warp_has_rows = __any_sync(0xffffffffU, real_row);
      const int plain_in_warp = __reduce_min_sync(0xffffffffU, real_row ? plain : 0x7fffffff);
      int key0 = (item.first + (kSplitKeys ? x : 0)) * kKeyTile + c * 64;

      float reference = -INFINITY;  // in units of the exponent, with the type's shift taken off
      float sum = 0.0f;
#pragma unroll 1
      for (int i = 0; i < count; ++i, key0 += (kSplitKeys ? 2 : 1) * kKeyTile) {
        ok = warp_wait(&sh.s_full[x], s_phase, abort_flag);
        if (!ok) break;
        s_phase ^= 1;
        tcgen05_fence_after();
        // the accumulator is complete up to the tile before this one, and this one's products wait for both warpgroups
        if ((i & (kKeepTiles - 1)) == 0 && i > 0 && warp_has_rows) {
          // In line or called, whichever leaves the loop its registers: long trees with heads of 64 164 us and 153, 4 x 4096 packed tokens 499
          // and 535 us; without this branch 153 and 495.
          float4* to = kept_at<kDim>(p.workspace, item.slot, x, c) + row;
          sum = kPaged ? keep_accumulator_call<kDim>(o_addr, to, &sh.kept[x][c][row], reference, sum, i > kKeepTiles)
                       : keep_accumulator<kDim>(o_addr, to, &sh.kept[x][c][row], reference, sum, i > kKeepTiles, false);
        }
        if (warp_has_rows) {
          float s[64];
          tmem_ld_32x32b_x32(s_addr, s);
          tmem_ld_32x32b_x32(s_addr + 32, s + 32);
          tmem_wait_ld();
          if (key0 + 64 > plain_in_warp) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int word0 = key0 + w * 32;
              const int seen = min(max(plain - word0, 0), 32);
              uint32_t bits = seen == 32 ? 0xffffffffU : (1u << seen) - 1u;
              if ((kPaged && p.mask != nullptr) && real_row && seen < 32) {
                const uint32_t* mask_row = p.mask + static_cast<long long>(item.token0 + (kSplitKeys ? 0 : x * tokens_per_half) + row_token) * p.mask_stride;
                const int node = word0 - item.prefix;  // of the word's first key; negative before the first drafted token
                const int word = node >> 5;
                // plain loads: the kernel in front, which may have written the mask, can still run when this one begins
                const uint32_t lo = word >= 0 && word < p.mask_words ? mask_row[word] : 0u;
                const uint32_t hi = word + 1 >= 0 && word + 1 < p.mask_words ? mask_row[word + 1] : 0u;
                bits |= __funnelshift_r(lo, hi, node & 31);
                const int there = min(max(item.keys - word0, 0), 32);
                if (there < 32) bits &= (1u << there) - 1u;
              }
#pragma unroll
              for (int e = 0; e < 32; ++e) s[w * 32 + e] = (bits >> e) & 1u ? s[w * 32 + e] : -INFINITY;
            }
          }
          float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int e = 4; e < 60; e += 8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) tops[j] = max3_f32(tops[j], s[e + 2 * j], s[e + 2 * j + 1]);
          }
          tops[0] = max3_f32(tops[0], s[60], s[61]);
          tops[1] = max3_f32(tops[1], s[62], s[63]);
          sh.row_max[x][c][row] = fmaxf(max3_f32(tops[0], tops[1], tops[2]), tops[3]) * p.scale_log2 - kShift<kBf16>;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.max_ready[x][quarter]);
          ok = warp_wait(&sh.max_ready[x][quarter], max_phase, abort_flag);
          if (!ok) break;
          max_phase ^= 1;
          const float top = fmaxf(sh.row_max[x][0][row], sh.row_max[x][1][row]);
          const bool moves = top > reference + kRescaleStep;  // true for the first key that is seen
          if (__any_sync(0xffffffffU, moves)) {
            // the reference moves for some row: its accumulator and sum shrink
            const float shrink = moves ? exp2_approx(reference - top) : 1.0f;  // 0 where nothing was seen before
            if (moves) reference = top;
            sum *= shrink;
            if (i > 0) {
#pragma unroll 1
              for (int d = 0; d < kDim / 2; d += 8) {
                float o[8];
                tmem_ld_32x32b_x8(o_addr + d, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] *= shrink;
                tmem_st_32x32b_x8(o_addr + d, o);
              }
            }
          }
          // The probabilities are rounded to 16 bits once, as an operand of the second product; the denominator adds up the numbers
          // before that, so that a row's roundings, of either sign, do not weigh on all of its values together.  A tile's 64 are added up
          // by themselves: one at a time, small numbers would be lost beside the sum of many keys.
          const float base = reference == -INFINITY ? 0.0f : reference;
          const unsigned long long scale2 = pack_f32x2(p.scale_log2, p.scale_log2), base2 = pack_f32x2(-base, -base);
          unsigned long long sum_a = pack_f32x2(0.0f, 0.0f), sum_b = pack_f32x2(0.0f, 0.0f);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t packed[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float lo, hi;
              unpack_f32x2(fma_f32x2(pack_f32x2(s[h * 32 + 2 * e], s[h * 32 + 2 * e + 1]), scale2, base2), lo, hi);
              if (by_polynomial<kDim, kSplitKeys>(e)) {
                lo = exp2_polynomial(lo);
                hi = exp2_polynomial(hi);
              } else {
                lo = exp2_approx(lo);
                hi = exp2_approx(hi);
              }
              if (e & 1) {
                sum_a = add_f32x2(sum_a, pack_f32x2(lo, hi));
              } else {
                sum_b = add_f32x2(sum_b, pack_f32x2(lo, hi));
              }
              packed[e] = pack16<kBf16>(lo, hi);
            }
            tmem_st_32x32b_x16(s_addr + h * 16, packed);
          }
          float lo, hi;
          unpack_f32x2(add_f32x2(sum_a, sum_b), lo, hi);
          sum += lo + hi;
          tmem_wait_st();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[x]);
      }
      if (!ok) break;

      // ------------------------------------------------------------- what leaves: normalised to the output, or a part
      // the accumulators are complete once all parts of the probabilities have been used
      const int n = item.end - item.first;
      const int count_a = kSplitKeys ? (n + 1) / 2 : count, count_b = kSplitKeys ? n / 2 : 0;
      if (count_a > 0) ok = warp_wait(&sh.o_full[kSplitKeys ? 0 : x], o_phase & 1, abort_flag);
      if (ok && count_b > 0) ok = warp_wait(&sh.o_full[1], (o_phase >> 1) & 1, abort_flag);
      if (!ok) break;
      if (count_a > 0) o_phase ^= 1;
      if (count_b > 0) o_phase ^= 2;
      const int parity = index & 1;
      if (count > kKeepTiles && warp_has_rows) {
        sum = keep_accumulator<kDim>(o_addr, kept_at<kDim>(p.workspace, item.slot, x, c) + row, &sh.kept[x][c][row], reference, sum, true, true);
      }
      sh.state[parity][x][c][row] = make_float2(reference, sum);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.state_full[kSplitKeys ? 0 : x]);
      ok = warp_wait(&sh.state_full[kSplitKeys ? 0 : x], parity, abort_flag);
      if (!ok) break;
      tcgen05_fence_after();
      float weight_a = 1.0f, weight_b = 0.0f;  // of the two sides' accumulators
      if (kSplitKeys) {
        const float2 a = sh.state[parity][0][0][row], b = sh.state[parity][1][0][row];
        reference = fmaxf(a.x, b.x);
        const float base = reference == -INFINITY ? 0.0f : reference;
        weight_a = exp2_approx(a.x - base);
        weight_b = exp2_approx(b.x - base);
        sum = (a.y + sh.state[parity][0][1][row].y) * weight_a + (b.y + sh.state[parity][1][1][row].y) * weight_b;
      } else {
        sum = sh.state[parity][x][0][row].y + sh.state[parity][x][1][row].y;
      }
      const int half = kSplitKeys ? 0 : x;
      const int slot = item.slot;
      const Parts parts = parts_of(p.workspace, gridDim.x);
      const size_t part = (static_cast<size_t>(blockIdx.x) * 2 + max(slot, 0)) * 2 + half;
      const int token = item.token0 + (kSplitKeys ? 0 : x * tokens_per_half) + row_token;
      const int head = item.kv_head * p.group + row - row_token * p.group;
      if (slot < 0) {
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        weight_a *= inverse;
        weight_b *= inverse;
      }
      if (warp_has_rows) {
        // the columns of this warpgroup: a half of the head dimension, or (kSplitKeys) a quarter, in chunks
        constexpr int kColumns = kSplitKeys ? kDim / 4 : kDim / 2, kChunk = 16;
        const int c_begin = (kSplitKeys ? group_index : c) * kColumns;
        const uint32_t o_a = tmem_base + lanes + kTmemO + half * kDim;
        uint16_t* out_row = p.out + token * p.out_token_stride + head * p.out_head_stride;
        if (!real_row) out_row = nullptr;
#pragma unroll 1
        for (int d = c_begin; d < c_begin + kColumns; d += kChunk) {
          float o[kChunk];
          if (count_a > 0) {
            tmem_ld_32x32b_x16(o_a + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < kChunk; ++e) o[e] *= weight_a;
          } else {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) o[e] = 0.0f;
          }
          if (kSplitKeys && count_b > 0) {
            float o_b[kChunk];
            tmem_ld_32x32b_x16(o_a + kDim + d, o_b);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < kChunk; ++e) o[e] = fmaf(o_b[e], weight_b, o[e]);
          }
          if (slot < 0) {
            // A lane has two pieces of 16 bytes of its row.  Two lanes trade one of theirs each, so that a store
            // instruction writes whole sectors of 16 rows instead of half sectors of 32.
            constexpr int kPieces = kChunk / 8;
            uint32_t piece[kPieces][4];
#pragma unroll
            for (int e = 0; e < kChunk / 2; ++e) piece[e / 4][e % 4] = pack16<kBf16>(o[2 * e], o[2 * e + 1]);
#pragma unroll
            for (int bit = 1; bit < kPieces; bit <<= 1) {
              const bool upper = (lane & bit) != 0;
#pragma unroll
              for (int i = 0; i < kPieces; ++i) {
                if (i & bit) continue;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                  const uint32_t got = __shfl_xor_sync(0xffffffffU, upper ? piece[i][w] : piece[i + bit][w], bit);
                  if (upper) {
                    piece[i][w] = got;
                  } else {
                    piece[i + bit][w] = got;
                  }
                }
              }
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
              uint16_t* to = reinterpret_cast<uint16_t*>(
                  __shfl_sync(0xffffffffU, reinterpret_cast<unsigned long long>(out_row), (lane & ~(kPieces - 1)) + i));
              if (to != nullptr) {
                *reinterpret_cast<uint4*>(to + d + (lane & (kPieces - 1)) * 8) = make_uint4(piece[i][0], piece[i][1], piece[i][2], piece[i][3]);
              }
            }
          } else if (real_row) {
            float4* to = parts.o + (part * (kDim / 4) + d / 4) * kRows + row;
#pragma unroll
            for (int e = 0; e < kChunk; e += 4) to[e / 4 * kRows] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (real_row && c == 0 && (!kSplitKeys || x == 0)) {
          if (slot >= 0) {
            parts.state[part * kRows + row] = make_float2(reference, sum);
          } else if (p.lse != nullptr) {
            p.lse[static_cast<long long>(token) * p.heads + head] =
                sum == 0.0f ? -INFINITY : (reference + log2f(sum)) * 0.69314718055994531f;
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.item_empty[slot_index]);
        if (kSplitKeys) {
          if (count_a > 0) mbar_arrive(&sh.o_empty[0]);
          if (count_b > 0) mbar_arrive(&sh.o_empty[1]);
        } else if (count > 0) {
          mbar_arrive(&sh.o_empty[x]);
        }
      }
    }
  }

  // ------------------------------------------------------------------- teardown
  tcgen05_fence_before();
  __syncthreads();
  if (sh.abort_flag != 0) {
    if (threadIdx.x == 0) atomicExch(p.status, FT_ERR_TIMEOUT);
    for (int i = 0; i < 64; ++i) __nanosleep(20000);  // copies in flight land before the shared memory is given up
    __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Adds up the parts of the row tiles that were split over CTAs: block (c, y) takes the row tile that begins in CTA c and
// does not end there.  A thread has four columns of one row; lanes run over rows first, as the parts are laid out.
constexpr int kCombineThreads = 256;
// Blocks per CTA.  Those of CTAs without such a row tile leave at once, but 148 x 8 of them cost about a microsecond; pairs have
// twice the rows.  B200: trees over 131072 and 65001 tokens (pairs) 194.5 us with 8, 191.4 with 16, 190.7 with 24; a prompt of
// 200 tokens (split) 10.9 with 4, 11.5 with 8, 12.7 with 16, one token over 1500 keys 12.9, 12.5 and 12.3.
template <bool kSplitKeys>
constexpr int kCombineBlocks = kSplitKeys ? 8 : 16;

template <int kDim, bool kBf16>
__global__ void __launch_bounds__(kCombineThreads) serve_attention_combine_kernel(const ServeAttentionParams p, int ctas, int halves) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Parts parts = parts_of(p.workspace, ctas);
  const int cta = blockIdx.x;
  const Unfinished u = parts.unfinished[cta];
  if (u.valid == 0) return;
  const int tokens_per_half = p.tokens_per_tile;
  const int lane = threadIdx.x & 31;
  constexpr int kColumnGroups = kDim / 16;  // a warp takes 8 rows x 4 x 4 columns
  for (int unit = blockIdx.y * (kCombineThreads / 32) + threadIdx.x / 32; unit < halves * (kRows / 8) * kColumnGroups;
       unit += gridDim.y * (kCombineThreads / 32)) {
    const int columns = (unit % kColumnGroups) * 4 + (lane >> 3);
    const int rows = unit / kColumnGroups;
    const int half = rows / (kRows / 8), row = rows % (kRows / 8) * 8 + (lane & 7);
    const int row_token = row / p.group, row_head = row - row_token * p.group;
    if (row_token >= tokens_per_half || half * tokens_per_half + row_token >= u.tokens) continue;
    // the first part lies in slot 1 of its CTA, the others in slot 0
    auto part_at = [&](int c) { return (static_cast<size_t>(c) * 2 + (c == cta ? 1 : 0)) * 2 + half; };
    float reference = -INFINITY, sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = cta; c <= u.last_cta; ++c) {
      const float2 state = parts.state[part_at(c) * kRows + row];
      const float4 add = parts.o[(part_at(c) * (kDim / 4) + columns) * kRows + row];
      const float next = fmaxf(reference, state.x), base = next == -INFINITY ? 0.0f : next;
      const float shrink = exp2_approx(reference - base), weight = exp2_approx(state.x - base);
      reference = next;
      sum = fmaf(state.y, weight, sum * shrink);
      o.x = fmaf(add.x, weight, o.x * shrink);
      o.y = fmaf(add.y, weight, o.y * shrink);
      o.z = fmaf(add.z, weight, o.z * shrink);
      o.w = fmaf(add.w, weight, o.w * shrink);
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const long long token = u.token0 + half * tokens_per_half + row_token;
    const int head = u.kv_head * p.group + row_head;
    *reinterpret_cast<uint2*>(p.out + token * p.out_token_stride + head * p.out_head_stride + columns * 4) =
        make_uint2(pack16<kBf16>(o.x * inverse, o.y * inverse), pack16<kBf16>(o.z * inverse, o.w * inverse));
    if (p.lse != nullptr && columns == 0) {
      p.lse[token * p.heads + head] = sum == 0.0f ? -INFINITY : (reference + log2f(sum)) * 0.69314718055994531f;
    }
  }
}

size_t serve_attention_workspace(int sm_count) { return parts_bytes(sm_count); }

template <int kDim, bool kBf16, bool kSplitKeys, bool kPaged>
static cudaError_t launch_form(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ServeAttentionParams& p, int sm_count,
                               cudaStream_t stream) {
  using L = Layout<kDim, kSplitKeys>;
  static std::atomic<unsigned long long> configured{0};  // a bit per device
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (device & 63);
  if (device > 63 || (configured.load(std::memory_order_relaxed) & bit) == 0) {
    err = cudaFuncSetAttribute(serve_attention_kernel<kDim, kBf16, kSplitKeys, kPaged>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (err != cudaSuccess) return err;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  // Both kernels may start while the one in front of them drains (they wait for its end before they touch memory).
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(sm_count);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = L::kBytes;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  err = cudaLaunchKernelEx(&config, serve_attention_kernel<kDim, kBf16, kSplitKeys, kPaged>, q, k, v, p);
  if (err != cudaSuccess) return err;
  config.gridDim = dim3(sm_count, kCombineBlocks<kSplitKeys>);
  config.blockDim = dim3(kCombineThreads);
  config.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&config, serve_attention_combine_kernel<kDim, kBf16>, p, sm_count, static_cast<int>(L::kQTiles));
}

template <int kDim, bool kBf16>
static cudaError_t launch_types(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ServeAttentionParams& p, bool split_keys,
                                int sm_count, cudaStream_t stream) {
  if (p.page_table != nullptr) {
    return split_keys ? launch_form<kDim, kBf16, true, true>(q, k, v, p, sm_count, stream) : launch_form<kDim, kBf16, false, true>(q, k, v, p, sm_count, stream);
  }
  return split_keys ? launch_form<kDim, kBf16, true, false>(q, k, v, p, sm_count, stream) : launch_form<kDim, kBf16, false, false>(q, k, v, p, sm_count, stream);
}

cudaError_t launch_serve_attention(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ServeAttentionParams& p, int dtype,
                                   bool split_keys, int sm_count, cudaStream_t stream) {
  if (dtype == FT_SRC_BF16) {
    return p.head_dim == 128 ? launch_types<128, true>(q, k, v, p, split_keys, sm_count, stream)
                             : launch_types<64, true>(q, k, v, p, split_keys, sm_count, stream);
  }
  return p.head_dim == 128 ? launch_types<128, false>(q, k, v, p, split_keys, sm_count, stream)
                           : launch_types<64, false>(q, k, v, p, split_keys, sm_count, stream);
}

}  // namespace ftg
