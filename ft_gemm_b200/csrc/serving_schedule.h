// How the attention over packed prompts and over the cache is cut into equal shares: plain integer arithmetic, the same
// on the device and on the host (where it is tested).
//
// A sequence of n queries and some keys makes, for each key head, ceil(n / tokens_per_item) row tiles; a row tile works
// through the 128-key tiles that any of its rows may see.  To begin and end a row tile costs about as much as kItemCost
// key tiles, so a row tile of T key tiles is T + kItemCost units of work, the first kItemCost of them without a key tile.
// The units of all row tiles, heads and sequences are numbered in a row, and CTA c takes [c * share, (c + 1) * share); a
// row tile whose first key tile lies in a share's front belongs to that share from its beginning.
#pragma once
#include <stdint.h>

// FT_HD_CALL: a function of its own in device code, where these steps stand beside loops that want the instruction cache.
#ifdef __CUDACC__
#define FT_HD __host__ __device__ __forceinline__
#define FT_HD_CALL static __host__ __device__ __noinline__
#else
#define FT_HD inline
#define FT_HD_CALL static inline
#endif

namespace ftg {

constexpr int kKeyTile = 128;
constexpr int kItemCost = 2;

// 64-bit numbers that nearly always fit into 32 bits, where a division is several times cheaper
FT_HD_CALL long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// sum over i in [0, n) of floor((a i + b) / m) for a, b >= 0, m > 0, in O(log) steps (the Euclid-like recursion on lattice
// points under a line)
FT_HD_CALL long long floor_sum(long long n, long long m, long long a, long long b) {
  long long total = 0;
  while (n > 0) {
    if (a >= m) {
      const long long whole = quotient(a, m);
      total += n * (n - 1) / 2 * whole;
      a -= whole * m;
    }
    if (b >= m) {
      const long long whole = quotient(b, m);
      total += n * whole;
      b -= whole * m;
    }
    const long long top = a * n + b;
    if (top < m) break;
    n = quotient(top, m);
    b = top - n * m;
    const long long t = m;
    m = a;
    a = t;
  }
  return total;
}

struct SequenceTiles {
  int queries, keys;    // keys: how many may be read
  int prefix;           // key tokens in front of the first query's own (negative: the first queries see nothing)
  int row_tiles;        // per key head
  int tokens_per_item;
  bool chain;           // query t sees keys [0, prefix + t]; otherwise row tiles count all keys
  bool ramp;            // row tiles are numbered with their own key limit; otherwise with all keys

  FT_HD static SequenceTiles make(int queries, int keys, int full_keys, int tokens_per_item, bool chain) {
    SequenceTiles s;
    s.queries = queries;
    s.keys = keys;
    s.prefix = full_keys - queries;
    s.tokens_per_item = tokens_per_item;
    s.row_tiles = queries <= 0 ? 0 : (queries - 1) / tokens_per_item + 1;
    s.chain = chain;
    s.ramp = chain && keys == full_keys;
    return s;
  }
  // how many leading keys the rows up to token `end` (exclusive) may see
  FT_HD int limit(int end) const {
    if (!chain) return keys;
    const int own = prefix + (end < queries ? end : queries);
    return own < 0 ? 0 : own < keys ? own : keys;
  }
  FT_HD static int tiles(int limit) { return limit <= 0 ? 1 : (limit - 1) / kKeyTile + 1; }
  // units of row tile r: at least one key tile, so that rows without keys are written too
  FT_HD int units_of(int r) const {
    if (!ramp) return tiles(keys) + kItemCost;
    const long long end = static_cast<long long>(r + 1) * tokens_per_item;
    return tiles(limit(end < queries ? static_cast<int>(end) : queries)) + kItemCost;
  }
  // units of the row tiles in front of r, r in [0, row_tiles]
  FT_HD long long units_before(int r) const { return units_before_of(*this, r); }
  FT_HD long long units_per_head() const { return row_tiles == 0 ? 0 : units_before(row_tiles); }
  FT_HD_CALL long long units_before_of(const SequenceTiles& t, int r) {
    if (!t.ramp) return static_cast<long long>(r) * (tiles(t.keys) + kItemCost);
    const int inner = r < t.row_tiles ? r : t.row_tiles - 1;  // the last row tile ends with the queries, not on the line
    long long empty = 0;                                  // row tiles that see nothing
    if (t.prefix < 0) {
      empty = quotient(t.tokens_per_item - t.prefix, t.tokens_per_item) - 1;
      empty = empty > inner ? inner : empty;
    }
    long long total = static_cast<long long>(inner) * kItemCost + empty +
                      floor_sum(inner - empty, kKeyTile, t.tokens_per_item, static_cast<long long>(t.tokens_per_item) * (empty + 1) + t.prefix + kKeyTile - 1);
    if (r == t.row_tiles && t.row_tiles > 0) total += t.units_of(t.row_tiles - 1);
    return total;
  }
};

}  // namespace ftg
