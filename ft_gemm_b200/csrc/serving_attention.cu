// Attention of each sequence's queries over its keys, packed one behind the other or in the pages of a cache:
//   o_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = exp(scale q_t k_j) over the keys j that token t sees.
//
// One persistent CTA per SM takes an equal share of the 128-key tiles of the whole call (serving_schedule.h), so the
// lengths of the sequences do not matter to the balance, and a long context is split over as many CTAs as there are when
// there are few rows.  The query heads of a key head are rows of one tile (row = token * group + head in group), which
// reads K and V once for the group.  Two warpgroups do the softmax, one thread per row, each on scores of its own:
//   kSplitKeys = false   two row tiles of 128 rows that share every K and V tile   (many rows)
//   kSplitKeys = true    one row tile; the warpgroups take the even and the odd key tiles and merge at the end   (few rows)
// While one warpgroup is in its softmax the tensor core works for the other: scores S = Q K^T into tensor memory, the
// probabilities go back to tensor memory in 16 bits over the scores they came from, and are the left operand of
// O += P V.  The exponent's reference follows the running maximum in steps of 2^8 only, so that the accumulator in
// tensor memory is hardly ever rescaled.
//
//   warp 0      walks the share: item descriptors for the others, tensor copies of Q, K and V
//   warp 1      issues the matrix instructions
//   warps 4-7, 8-11   softmax of A and B, and what leaves the kernel
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

constexpr int kRows = 128;  // rows of a tile: the lanes of tensor memory
constexpr int kThreads = 384;
// setmaxnreg.inc waits for registers of the CTA's own allotment (384 x 168): the three numbers have to fit together.
constexpr int kLaunchRegs = 168, kIssueRegs = 72, kSoftmaxRegs = 216;
static_assert(128 * kIssueRegs + 256 * kSoftmaxRegs <= kThreads * kLaunchRegs, "setmaxnreg.inc would wait for registers the CTA does not own");
constexpr uint64_t kTimeoutNs = 2000000000ull;
constexpr float kRescaleStep = 8.0f;  // log2 units
constexpr int kItems = 4;             // descriptors in flight
constexpr int kMaxStages = 12;
constexpr uint32_t kTmemS = 0, kTmemO = 256;  // S of A and B: 128 columns each; O of A and B: kDim each

struct Item {
  int sequence;
  int token0;      // first query row in q and out
  int tokens;      // queries of this row tile; negative: the walk is over
  int place0;      // place of the first query among the sequence's queries
  int kv_head;
  int key_row0;    // packed keys: row of the first key
  int prefix, keys, limit;  // limit: no row sees a key at or behind it
  int first, end;  // key tiles of this part
  int slot;        // -1: the whole row tile, straight to the output; otherwise which part in the workspace
};

struct Shared {
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_full[2], o_full[2], o_empty[2];
  uint64_t item_full[kItems], item_empty[kItems];
  Item items[kItems];
  uint32_t tmem_base;
  int abort_flag;
  long long scan[kThreads / 32];
  int start_sequence;
  long long start_tile;
  uint64_t state_full;  // kSplitKeys: both warpgroups have written their state
};

// kSplitKeys, behind Shared: {reference, sum} of each warpgroup's rows, in turn for odd and even items.
typedef float2 SharedState[2][2][kRows];

template <int kDim, bool kSplitKeys>
struct Layout {
  static constexpr int kSlabs = kDim / 64;              // 128-byte columns of a row of Q, K or V
  static constexpr int kTileBytes = kSlabs * 128 * 128;
  static constexpr int kQTiles = kSplitKeys ? 1 : 2;
  static constexpr int kStages = kDim == 64 ? 10 : 5;
  static constexpr int kBytes = (kQTiles + kStages) * kTileBytes + static_cast<int>(sizeof(Shared)) +
                                (kSplitKeys ? static_cast<int>(sizeof(SharedState)) : 0) + 1024;
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

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffU, mbar_wait_bounded(bar, parity, abort_flag, kTimeoutNs));
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
// D[tmem] (+)= A[tmem] * B[smem], 16-bit operands; A holds two elements per column.
__device__ __forceinline__ void umma_f16_tmem_a(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// V as the right operand: 64 elements of a row (one swizzled 128-byte column) are contiguous along N, keys along K.
// Leading byte offset: from one 64-element column to the next (128 rows of 128 bytes); stride byte offset: 8 keys.
__device__ __forceinline__ uint64_t make_smem_desc_sw128_mn(uint32_t smem_addr) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((smem_addr >> 4) & 0x3fff);
  desc |= static_cast<uint64_t>((128 * 128) >> 4) << 16;
  desc |= static_cast<uint64_t>(1024 >> 4) << 32;
  desc |= static_cast<uint64_t>(1) << 46;
  desc |= static_cast<uint64_t>(2) << 61;
  return desc;
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
template <int Regs>
__device__ __forceinline__ void reg_release() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs));
}
template <int Regs>
__device__ __forceinline__ void reg_acquire() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs));
}

// What the call's arrays say about sequence b, cut to what may be read.
struct Sequence {
  int token0, key_row0;
  SequenceTiles tiles;
};
__device__ __forceinline__ Sequence load_sequence(const ServeAttentionParams& p, int b, int tokens_per_item) {
  Sequence s;
  s.token0 = min(max(p.q_offsets[b], 0), p.query_tokens);
  const int queries = min(max(p.q_offsets[b + 1], s.token0), p.query_tokens) - s.token0;
  int keys, full;
  if (p.page_table != nullptr) {
    s.key_row0 = 0;
    full = max(p.lengths[b], 0);
    keys = min(full, p.table_pages * p.page_size);
  } else {
    s.key_row0 = min(max(p.k_offsets[b], 0), p.key_tokens);
    keys = full = min(max(p.k_offsets[b + 1], s.key_row0), p.key_tokens) - s.key_row0;
  }
  s.tiles = SequenceTiles::make(queries, keys, full, tokens_per_item, p.causal != 0 && p.mask == nullptr);
  return s;
}

// The queries of warpgroup `half` and the key tiles it works through.
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

template <int kDim, bool kBf16, bool kSplitKeys>
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
  SharedState& state = *reinterpret_cast<SharedState*>(&sh + 1);
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tokens_per_half = kRows / p.group;
  const int tokens_per_item = L::kQTiles * tokens_per_half;
  const bool chain = p.causal != 0 && p.mask == nullptr;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.state_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], kSplitKeys ? 8 : 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_empty[i], 9);
    }
    sh.abort_flag = 0;
    sh.start_sequence = -1;
    fence_barrier_init();
    prefetch_tensormap(&tmap_q);
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }

  // ---- this CTA's share: the key tiles of all sequences are summed by the whole CTA
  const int per_thread = (p.batch + kThreads - 1) / kThreads;
  const int scan_begin = min(static_cast<int>(threadIdx.x) * per_thread, p.batch), scan_end = min(scan_begin + per_thread, p.batch);
  long long mine = 0;
  for (int b = scan_begin; b < scan_end; ++b) mine += load_sequence(p, b, tokens_per_item).tiles.tiles_per_head() * p.kv_heads;
  long long before = mine;  // inclusive prefix within the warp
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long other = __shfl_up_sync(0xffffffffU, before, off);
    if (lane >= off) before += other;
  }
  if (lane == 31) sh.scan[warp] = before;
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  long long total = 0, front = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) front += sh.scan[w];
    total += sh.scan[w];
  }
  before += front - mine;
  const long long share = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(p.min_share));
  const long long share_begin = min(share * blockIdx.x, total), share_end = min(share_begin + share, total);
  if (share_begin < share_end && before <= share_begin && share_begin < before + mine) {
    long long at = before;
    for (int b = scan_begin; b < scan_end; ++b) {
      const long long here = load_sequence(p, b, tokens_per_item).tiles.tiles_per_head() * p.kv_heads;
      if (share_begin < at + here) {
        sh.start_sequence = b;
        sh.start_tile = share_begin - at;
        break;
      }
      at += here;
    }
  }
  __syncthreads();
  const uint32_t tmem_base = sh.tmem_base;

  if (warp < 4) {
    reg_release<kIssueRegs>();
    if (warp == 0) {
      // ------------------------------------------------------------- the walk, and the tensor copies
      Unfinished unfinished = {};
      int stage = 0, stage_phase = 0, q_phase = 0;
      uint32_t item_index = 0;
      bool ok = true;
      long long left = share_end - share_begin;
      int b = sh.start_sequence;
      Sequence seq = {};
      int kv_head = 0, row_tile = 0, first = 0, row_tiles_count = 0;
      if (left > 0) {
        seq = load_sequence(p, b, tokens_per_item);
        const long long per_head = seq.tiles.tiles_per_head();
        const long long at = sh.start_tile;
        kv_head = static_cast<int>(at / per_head);
        const long long inner = at - kv_head * per_head;
        int lo = 0, hi = seq.tiles.row_tiles;  // tiles_before(lo) <= inner < tiles_before(hi)
        while (hi - lo > 1) {
          const int step = (hi - lo + 31) / 32;
          const int probe = min(lo + lane * step, hi);
          const int below = __popc(__ballot_sync(0xffffffffU, seq.tiles.tiles_before(probe) <= inner && probe < hi));
          lo = lo + (below - 1) * step;
          hi = min(lo + step, hi);
        }
        row_tile = lo;
        first = static_cast<int>(inner - seq.tiles.tiles_before(lo));
      }
      while (ok) {
        const int slot_index = item_index % kItems;
        ok = warp_wait(&sh.item_empty[slot_index], ((item_index / kItems) & 1) ^ 1, abort_flag);
        if (!ok) break;
        Item item = {};
        if (left <= 0) {
          item.tokens = -1;
          if (lane == 0) {
            sh.items[slot_index] = item;
            mbar_arrive(&sh.item_full[slot_index]);
          }
          break;
        }
        row_tiles_count = seq.tiles.tiles_of(row_tile);
        const int end = static_cast<int>(min(static_cast<long long>(row_tiles_count), first + left));
        item.sequence = b;
        item.place0 = row_tile * tokens_per_item;
        item.token0 = seq.token0 + item.place0;
        item.tokens = min(seq.tiles.queries - item.place0, tokens_per_item);
        item.kv_head = kv_head;
        item.key_row0 = seq.key_row0;
        item.prefix = seq.tiles.prefix;
        item.keys = seq.tiles.keys;
        item.limit = seq.tiles.limit(item.place0 + item.tokens);
        const int real = item.limit <= 0 ? 0 : (item.limit - 1) / kKeyTile + 1;  // a numbered tile may have nothing in it
        item.first = min(first, real);
        item.end = min(end, real);
        item.slot = first == 0 && end == row_tiles_count ? -1 : first > 0 ? 0 : 1;
        if (first == 0 && end < row_tiles_count) {
          unfinished.valid = 1;
          unfinished.last_cta = blockIdx.x + static_cast<int>((row_tiles_count - end + share - 1) / share);
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
          auto load = [&](const CUtensorMap* map, int tile) -> bool {
            if (!warp_wait(&sh.kv_empty[stage], stage_phase ^ 1, abort_flag)) return false;
            uint8_t* to = smem_kv + stage * L::kTileBytes;
            if (p.page_table == nullptr) {
              if (lane == 0) {
                mbar_arrive_expect_tx(&sh.kv_full[stage], L::kTileBytes);
#pragma unroll
                for (int sl = 0; sl < L::kSlabs; ++sl) {
                  tma_load_3d(to + sl * (128 * 128), map, &sh.kv_full[stage], 64 * sl, kv_head, item.key_row0 + tile * kKeyTile);
                }
              }
            } else {
              const int box = min(p.page_size, kKeyTile);
              const int boxes = (min(item.limit - tile * kKeyTile, kKeyTile) + box - 1) / box;  // behind the limit nothing is read
              if (lane == 0) mbar_arrive_expect_tx(&sh.kv_full[stage], boxes * box * L::kSlabs * 128);
              __syncwarp();
              if (lane < boxes) {
                const int key = tile * kKeyTile + lane * box;
                int page = p.page_table[static_cast<long long>(b) * p.table_stride + key / p.page_size];
                if (page < 0 || page > p.pages) page = p.pages;  // outside the tensor: filled with zeros
#pragma unroll
                for (int sl = 0; sl < L::kSlabs; ++sl) {
                  tma_load_4d(to + sl * (128 * 128) + lane * box * 128, map, &sh.kv_full[stage], 64 * sl, key % p.page_size, kv_head, page);
                }
              }
            }
            if (++stage == L::kStages) {
              stage = 0;
              stage_phase ^= 1;
            }
            return true;
          };
          ok = load(&tmap_k, item.first);
          for (int t = item.first; ok && t < item.end; ++t) {
            if (kSplitKeys) {
              if (t + 1 < item.end) ok = load(&tmap_k, t + 1);
              if (ok) ok = load(&tmap_v, t);
            } else {
              ok = load(&tmap_v, t);
              if (ok && t + 1 < item.end) ok = load(&tmap_k, t + 1);
            }
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
              seq = load_sequence(p, ++b, tokens_per_item);
            } while (seq.tiles.row_tiles == 0 && b + 1 < p.batch);
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
      // ------------------------------------------------------------- matrix instructions
      constexpr uint32_t kIdescS = idesc16<kBf16>(128, false), kIdescO = idesc16<kBf16>(kDim, true);
      int stage = 0, stage_phase = 0, q_phase = 0;
      uint32_t p_phase[2] = {0, 0}, o_phase[2] = {0, 0};
      bool ok = true;
      const uint32_t q_addr = smem_u32(smem_q), kv_addr = smem_u32(smem_kv);

      auto issue_s = [&](int x, int k_stage) {
        const uint64_t a = make_smem_desc_sw128(q_addr + (kSplitKeys ? 0 : x) * L::kTileBytes), bd = make_smem_desc_sw128(kv_addr + k_stage * L::kTileBytes);
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k) {
          const int at = (k / 4) * ((128 * 128) >> 4) + (k % 4) * 2;
          umma_f16(tmem_base + kTmemS + x * 128, a + at, bd + at, kIdescS, k > 0);
        }
        umma_commit(&sh.s_full[x]);
      };
      auto issue_o = [&](int x, int v_stage, int steps, bool fresh) {
        const uint64_t bd = make_smem_desc_sw128_mn(kv_addr + v_stage * L::kTileBytes);
        for (int k = 0; k < steps; ++k) {
          umma_f16_tmem_a(tmem_base + kTmemO + x * kDim, tmem_base + kTmemS + x * 128 + k * 8, bd + k * (16 * 128 >> 4), kIdescO, !fresh || k > 0);
        }
      };
      auto next_stage = [&]() {
        if (++stage == L::kStages) {
          stage = 0;
          stage_phase ^= 1;
        }
      };
      // V rows behind the last key anyone sees hold whatever memory holds; their probabilities are zero, but zero times
      // NaN is not, so the instruction stops at the next multiple of 16 keys and the rows up to there are cleared.
      auto clear_v_tail = [&](int v_stage, int valid) {
        uint8_t* v = smem_kv + v_stage * L::kTileBytes;
        const int upto = (valid + 15) / 16 * 16;
        for (int i = lane; i < (upto - valid) * L::kSlabs * 8; i += 32) {
          const int row = valid + i / (L::kSlabs * 8), chunk = i % (L::kSlabs * 8);
          *reinterpret_cast<uint4*>(v + (chunk / 8) * (128 * 128) + row * 128 + (chunk % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_shared();
        __syncwarp();
      };

      for (uint32_t index = 0; ok; ++index) {
        const int slot_index = index % kItems;
        ok = warp_wait(&sh.item_full[slot_index], (index / kItems) & 1, abort_flag);
        if (!ok) break;
        const Item item = sh.items[slot_index];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.item_empty[slot_index]);
        if (item.tokens < 0) break;
        const int n = item.end - item.first;
        if (n <= 0) continue;
        const int count[2] = {HalfWork<kSplitKeys>(item, 0, tokens_per_half, chain).count, HalfWork<kSplitKeys>(item, 1, tokens_per_half, chain).count};
        ok = warp_wait(&sh.q_full, q_phase, abort_flag);
        if (!ok) break;
        q_phase ^= 1;

        // O += P V of warpgroup x for the key tile in v_stage, its i-th
        auto accumulate = [&](int x, int i, int v_stage, int steps) -> bool {
          if (i == 0) {
            if (!warp_wait(&sh.o_empty[x], o_phase[x] ^ 1, abort_flag)) return false;
            o_phase[x] ^= 1;
          }
          if (!warp_wait(&sh.p_full[x], p_phase[x], abort_flag)) return false;
          p_phase[x] ^= 1;
          tcgen05_fence_after();
          if (elect_one()) {
            issue_o(x, v_stage, steps, i == 0);
            if (i + 1 == count[x]) umma_commit(&sh.o_full[x]);
          }
          __syncwarp();
          return true;
        };
        auto valid_keys = [&](int tile) { return min(item.limit - tile * kKeyTile, kKeyTile); };

        if (kSplitKeys) {
          for (int t = 0; ok && t < min(n, 2); ++t) {
            ok = warp_wait(&sh.kv_full[stage], stage_phase, abort_flag);
            if (!ok) break;
            tcgen05_fence_after();
            if (elect_one()) {
              issue_s(t, stage);
              umma_commit(&sh.kv_empty[stage]);
              if (t + 1 == n) umma_commit(&sh.q_empty);
            }
            __syncwarp();
            next_stage();
          }
          for (int t = 0; ok && t < n; ++t) {
            const int x = t & 1;
            ok = warp_wait(&sh.kv_full[stage], stage_phase, abort_flag);
            if (!ok) break;
            const int valid = valid_keys(item.first + t);
            if (valid < kKeyTile) clear_v_tail(stage, valid);
            ok = accumulate(x, t >> 1, stage, (valid + 15) / 16);
            if (!ok) break;
            if (elect_one()) umma_commit(&sh.kv_empty[stage]);
            __syncwarp();
            next_stage();
            if (t + 2 < n) {
              ok = warp_wait(&sh.kv_full[stage], stage_phase, abort_flag);
              if (!ok) break;
              tcgen05_fence_after();
              if (elect_one()) {
                issue_s(x, stage);
                umma_commit(&sh.kv_empty[stage]);
                if (t + 3 == n) umma_commit(&sh.q_empty);
              }
              __syncwarp();
              next_stage();
            }
          }
        } else {
          ok = warp_wait(&sh.kv_full[stage], stage_phase, abort_flag);
          if (!ok) break;
          tcgen05_fence_after();
          if (elect_one()) {
            if (count[0] > 0) issue_s(0, stage);
            if (count[1] > 0) issue_s(1, stage);
            umma_commit(&sh.kv_empty[stage]);
            if (n == 1) umma_commit(&sh.q_empty);
          }
          __syncwarp();
          next_stage();
          for (int j = 0; ok && j < n; ++j) {
            const int v_stage = stage;
            ok = warp_wait(&sh.kv_full[stage], stage_phase, abort_flag);
            if (!ok) break;
            next_stage();
            const int k_stage = stage, k_phase = stage_phase;
            bool have_k = false;
            if (j + 1 < n) next_stage();
            const int valid = valid_keys(item.first + j);
            if (valid < kKeyTile) clear_v_tail(v_stage, valid);
            for (int x = 0; ok && x < 2; ++x) {
              if (j >= count[x]) continue;
              ok = accumulate(x, j, v_stage, (valid + 15) / 16);
              if (ok && j + 1 < count[x]) {
                if (!have_k) ok = warp_wait(&sh.kv_full[k_stage], k_phase, abort_flag);
                have_k = true;
                if (!ok) break;
                tcgen05_fence_after();
                if (elect_one()) issue_s(x, k_stage);
                __syncwarp();
              }
            }
            if (!ok) break;
            if (elect_one()) {
              umma_commit(&sh.kv_empty[v_stage]);
              if (j + 1 < n) umma_commit(&sh.kv_empty[k_stage]);
              if (j + 2 == n) umma_commit(&sh.q_empty);
            }
            __syncwarp();
          }
        }
      }
    }
  } else {
    // --------------------------------------------------------------- softmax: one thread per row
    reg_acquire<kSoftmaxRegs>();
    const int x = (warp - 4) >> 2;            // warpgroup A or B
    const int quarter = warp & 3;             // the lanes of tensor memory this warp can reach
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter) << 21;  // lane index in bits 16 and up, 32 lanes per warp
    const uint32_t s_addr = tmem_base + lanes + kTmemS + x * 128, o_addr = tmem_base + lanes + kTmemO + x * kDim;
    const int row_token = row / p.group, row_head = row - row_token * p.group;
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    const Parts parts = parts_of(p.workspace, gridDim.x);

    for (uint32_t index = 0; ok; ++index) {
      const int slot_index = index % kItems;
      ok = warp_wait(&sh.item_full[slot_index], (index / kItems) & 1, abort_flag);
      if (!ok) break;
      const Item item = sh.items[slot_index];
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_empty[slot_index]);
      if (item.tokens < 0) break;
      const HalfWork<kSplitKeys> work(item, x, tokens_per_half, chain);
      const bool real_row = row_token < min(work.tokens, tokens_per_half);
      const bool warp_has_rows = __any_sync(0xffffffffU, real_row);
      const int place = item.place0 + work.place0 + row_token;  // among the sequence's queries
      const long long token = item.token0 + work.place0 + row_token;
      // every key below `plain` is seen; with a mask its bits say which of the rest are
      const int plain = !real_row ? 0 : p.mask != nullptr ? min(item.prefix, item.keys) : chain ? min(item.limit, item.prefix + place + 1) : item.keys;
      const uint32_t* mask_row = p.mask != nullptr && real_row ? p.mask + token * p.mask_stride : nullptr;
      const int plain_in_warp = __reduce_min_sync(0xffffffffU, real_row ? plain : 0x7fffffff);

      float reference = -INFINITY;  // in units of the exponent, with the type's shift taken off
      float sum = 0.0f;
      for (int i = 0; i < work.count; ++i) {
        const int key0 = (item.first + (kSplitKeys ? 2 * i + x : i)) * kKeyTile;
        ok = warp_wait(&sh.s_full[x], s_phase, abort_flag);
        if (!ok) break;
        s_phase ^= 1;
        tcgen05_fence_after();
        if (warp_has_rows) {
          float s[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s + c * 32);
          tmem_wait_ld();
          if (key0 + kKeyTile > plain_in_warp) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int word0 = key0 + w * 32;
              const int seen = min(max(plain - word0, 0), 32);
              uint32_t bits = seen == 32 ? 0xffffffffU : (1u << seen) - 1u;
              if (mask_row != nullptr && seen < 32) {
                const int node = word0 - item.prefix;  // of the word's first key; negative before the first drafted token
                const int word = node >> 5;
                const uint32_t lo = word >= 0 && word < p.mask_words ? __ldg(mask_row + word) : 0u;
                const uint32_t hi = word + 1 >= 0 && word + 1 < p.mask_words ? __ldg(mask_row + word + 1) : 0u;
                bits |= __funnelshift_r(lo, hi, node & 31);
                const int there = min(max(item.keys - word0, 0), 32);
                if (there < 32) bits &= (1u << there) - 1u;
              }
#pragma unroll
              for (int e = 0; e < 32; ++e) s[w * 32 + e] = (bits >> e) & 1u ? s[w * 32 + e] : -INFINITY;
            }
          }
          float top_a = s[0], top_b = s[1];
#pragma unroll
          for (int e = 2; e < 126; e += 4) {
            top_a = max3_f32(top_a, s[e], s[e + 1]);
            top_b = max3_f32(top_b, s[e + 2], s[e + 3]);
          }
          const float top = max3_f32(top_a, top_b, fmaxf(s[126], s[127])) * p.scale_log2 - kShift<kBf16>;
          const bool moves = top > reference + kRescaleStep;  // true for the first key that is seen
          if (__any_sync(0xffffffffU, moves)) {
            const float next = moves ? top : reference;
            const float shrink = moves ? exp2_approx(reference - next) : 1.0f;  // 0 where nothing was seen before
            reference = next;
            sum *= shrink;
            if (i > 0) {
#pragma unroll 1
              for (int c = 0; c < kDim / 32; ++c) {
                float o[32];
                tmem_ld_32x32b_x32(o_addr + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= shrink;
                tmem_st_32x32b_x32(o_addr + c * 32, o);
              }
            }
          }
          const float base = reference == -INFINITY ? 0.0f : reference;
          const unsigned long long scale2 = pack_f32x2(p.scale_log2, p.scale_log2), base2 = pack_f32x2(-base, -base);
          unsigned long long sum_a = pack_f32x2(sum, 0.0f), sum_b = pack_f32x2(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t packed[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float lo, hi;
              unpack_f32x2(fma_f32x2(pack_f32x2(s[c * 32 + 2 * e], s[c * 32 + 2 * e + 1]), scale2, base2), lo, hi);
              lo = exp2_approx(lo);
              hi = exp2_approx(hi);
              if (e & 1) {
                sum_a = add_f32x2(sum_a, pack_f32x2(lo, hi));
              } else {
                sum_b = add_f32x2(sum_b, pack_f32x2(lo, hi));
              }
              packed[e] = pack16<kBf16>(lo, hi);
            }
            tmem_st_32x32b_x16(s_addr + c * 16, packed);
          }
          float lo, hi;
          unpack_f32x2(add_f32x2(sum_a, sum_b), lo, hi);
          sum = lo + hi;
          tmem_wait_st();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[x]);
      }
      if (!ok) break;

      // ------------------------------------------------------------- what leaves: normalised to the output, or a part
      float weight_a = 1.0f, weight_b = 0.0f;  // kSplitKeys: of the two warpgroups' sums
      int count_a = work.count, count_b = 0;
      if (kSplitKeys) {
        // two copies in turn: whoever writes the next but one has seen that all have read this one
        state[index & 1][x][row] = make_float2(reference, sum);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.state_full);
        ok = warp_wait(&sh.state_full, index & 1, abort_flag);
        if (!ok) break;
        const float2 a = state[index & 1][0][row], bs = state[index & 1][1][row];
        reference = fmaxf(a.x, bs.x);
        const float base = reference == -INFINITY ? 0.0f : reference;
        weight_a = exp2_approx(a.x - base);
        weight_b = exp2_approx(bs.x - base);
        sum = a.y * weight_a + bs.y * weight_b;
        const int n = item.end - item.first;
        count_a = (n + 1) / 2;
        count_b = n / 2;
        // both accumulators are read by both warpgroups, half of the columns each
        if (count_a > 0) ok = warp_wait(&sh.o_full[0], o_phase & 1, abort_flag);
        if (ok && count_b > 0) ok = warp_wait(&sh.o_full[1], (o_phase >> 1) & 1, abort_flag);
        if (!ok) break;
        if (count_a > 0) o_phase ^= 1;
        if (count_b > 0) o_phase ^= 2;
      } else if (work.count > 0) {
        ok = warp_wait(&sh.o_full[x], o_phase, abort_flag);
        if (!ok) break;
        o_phase ^= 1;
      }
      tcgen05_fence_after();
      const int half = kSplitKeys ? 0 : x;
      const size_t part = (static_cast<size_t>(blockIdx.x) * 2 + max(item.slot, 0)) * 2 + half;
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (kSplitKeys && item.slot < 0) {
        weight_a *= inverse;
        weight_b *= inverse;
      } else if (item.slot < 0) {
        weight_a = inverse;
      }
      if (warp_has_rows) {
        constexpr int kChunk = 32;
        const int c_begin = kSplitKeys ? x * (kDim / 2) : 0, c_end = kSplitKeys ? c_begin + kDim / 2 : kDim;
        const uint32_t o_a = tmem_base + lanes + kTmemO + half * kDim;
        uint16_t* out_row = p.out + token * p.out_token_stride + (static_cast<long long>(item.kv_head) * p.group + row_head) * p.out_head_stride;
#pragma unroll 1
        for (int c = c_begin; c < c_end; c += kChunk) {
          float o[kChunk];
          if (count_a > 0) {
            tmem_ld_32x32b_x32(o_a + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < kChunk; ++e) o[e] *= weight_a;
          } else {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) o[e] = 0.0f;
          }
          if (kSplitKeys && count_b > 0) {
            float o_b[kChunk];
            tmem_ld_32x32b_x32(o_a + kDim + c, o_b);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < kChunk; ++e) o[e] = fmaf(o_b[e], weight_b, o[e]);
          }
          if (real_row) {
            if (item.slot < 0) {
#pragma unroll
              for (int e = 0; e < kChunk; e += 8) {
                *reinterpret_cast<uint4*>(out_row + c + e) = make_uint4(pack16<kBf16>(o[e], o[e + 1]), pack16<kBf16>(o[e + 2], o[e + 3]),
                                                                        pack16<kBf16>(o[e + 4], o[e + 5]), pack16<kBf16>(o[e + 6], o[e + 7]));
              }
            } else {
              float4* to = parts.o + (part * (kDim / 4) + c / 4) * kRows + row;
#pragma unroll
              for (int e = 0; e < kChunk; e += 4) to[e / 4 * kRows] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        if (real_row && (!kSplitKeys || x == 0)) {
          if (item.slot >= 0) {
            parts.state[part * kRows + row] = make_float2(reference, sum);
          } else if (p.lse != nullptr) {
            p.lse[token * p.heads + item.kv_head * p.group + row_head] = sum == 0.0f ? -INFINITY : (reference + log2f(sum)) * 0.69314718055994531f;
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kSplitKeys) {
          if (count_a > 0) mbar_arrive(&sh.o_empty[0]);
          if (count_b > 0) mbar_arrive(&sh.o_empty[1]);
        } else if (work.count > 0) {
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
constexpr int kCombineBlocks = 4, kCombineThreads = 256;

template <int kDim, bool kBf16>
__global__ void __launch_bounds__(kCombineThreads) serve_attention_combine_kernel(const ServeAttentionParams p, int ctas, int halves) {
  const Parts parts = parts_of(p.workspace, ctas);
  const int cta = blockIdx.x;
  const Unfinished u = parts.unfinished[cta];
  if (u.valid == 0) return;
  const int tokens_per_half = kRows / p.group;
  const int lane = threadIdx.x & 31;
  constexpr int kColumnGroups = kDim / 16;  // a warp takes 8 rows x 4 x 4 columns
  for (int unit = blockIdx.y * (kCombineThreads / 32) + threadIdx.x / 32; unit < halves * (kRows / 8) * kColumnGroups;
       unit += kCombineBlocks * (kCombineThreads / 32)) {
    const int columns = (unit % kColumnGroups) * 4 + (lane >> 3);
    const int rows = unit / kColumnGroups;
    const int half = rows / (kRows / 8), row = rows % (kRows / 8) * 8 + (lane & 7);
    const int row_token = row / p.group, row_head = row - row_token * p.group;
    if (row_token >= tokens_per_half || half * tokens_per_half + row_token >= u.tokens) continue;
    // the first part lies in slot 1 of its CTA, the others in slot 0
    auto part_at = [&](int c) { return (static_cast<size_t>(c) * 2 + (c == cta ? 1 : 0)) * 2 + half; };
    float reference = -INFINITY;
    for (int c = cta; c <= u.last_cta; ++c) reference = fmaxf(reference, parts.state[part_at(c) * kRows + row].x);
    const float base = reference == -INFINITY ? 0.0f : reference;
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = cta; c <= u.last_cta; ++c) {
      const float2 state = parts.state[part_at(c) * kRows + row];
      const float4 add = parts.o[(part_at(c) * (kDim / 4) + columns) * kRows + row];
      const float weight = exp2_approx(state.x - base);
      sum = fmaf(state.y, weight, sum);
      o.x = fmaf(add.x, weight, o.x);
      o.y = fmaf(add.y, weight, o.y);
      o.z = fmaf(add.z, weight, o.z);
      o.w = fmaf(add.w, weight, o.w);
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

template <int kDim, bool kBf16, bool kSplitKeys>
static cudaError_t launch_form(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ServeAttentionParams& p, int sm_count,
                               cudaStream_t stream) {
  using L = Layout<kDim, kSplitKeys>;
  static std::atomic<unsigned long long> configured{0};  // a bit per device
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (device & 63);
  if (device > 63 || (configured.load(std::memory_order_relaxed) & bit) == 0) {
    err = cudaFuncSetAttribute(serve_attention_kernel<kDim, kBf16, kSplitKeys>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (err != cudaSuccess) return err;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  serve_attention_kernel<kDim, kBf16, kSplitKeys><<<sm_count, kThreads, L::kBytes, stream>>>(q, k, v, p);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  serve_attention_combine_kernel<kDim, kBf16><<<dim3(sm_count, kCombineBlocks), kCombineThreads, 0, stream>>>(p, sm_count, L::kQTiles);
  return cudaGetLastError();
}

template <int kDim, bool kBf16>
static cudaError_t launch_types(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ServeAttentionParams& p, bool split_keys,
                                int sm_count, cudaStream_t stream) {
  return split_keys ? launch_form<kDim, kBf16, true>(q, k, v, p, sm_count, stream) : launch_form<kDim, kBf16, false>(q, k, v, p, sm_count, stream);
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
