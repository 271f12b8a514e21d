// How the attention over packed prompts and over the cache is cut into equal shares: plain integer arithmetic, the same
// on the device and on the host (where it is tested).
//
// A sequence of n queries and some keys makes, for each key head, ceil(n / tokens_per_item) row tiles; a row tile works
// through the 128-key tiles that any of its rows may see.  All key tiles of all row tiles, heads and sequences in a row
// are numbered from 0 to W - 1, and CTA c takes [c * share, (c + 1) * share).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FT_HD __host__ __device__ __forceinline__
#else
#define FT_HD inline
#endif

namespace ftg {

constexpr int kKeyTile = 128;

// sum over i in [0, n) of floor((a i + b) / m) for a, b >= 0, m > 0, in O(log) steps (the Euclid-like recursion on lattice
// points under a line)
FT_HD long long floor_sum(long long n, long long m, long long a, long long b) {
  long long total = 0;
  while (n > 0) {
    if (a >= m) {
      total += n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      total += n * (b / m);
      b %= m;
    }
    const long long top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
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
    s.row_tiles = queries / tokens_per_item + (queries % tokens_per_item != 0 ? 1 : 0);
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
  // row tile r: at least 1, so that rows without keys are written too
  FT_HD int tiles_of(int r) const {
    if (!ramp) return tiles(keys);
    const long long end = static_cast<long long>(r + 1) * tokens_per_item;
    return tiles(limit(end < queries ? static_cast<int>(end) : queries));
  }
  // key tiles of the row tiles in front of r, r in [0, row_tiles]
  FT_HD long long tiles_before(int r) const {
    if (!ramp) return static_cast<long long>(r) * tiles(keys);
    const int inner = r < row_tiles ? r : row_tiles - 1;  // the last row tile ends with the queries, not on the line
    long long empty = (1 - static_cast<long long>(prefix) + tokens_per_item - 1) / tokens_per_item - 1;  // row tiles that see nothing
    if (prefix >= 1) empty = 0;
    empty = empty < 0 ? 0 : empty > inner ? inner : empty;
    long long total = empty + floor_sum(inner - empty, kKeyTile, tokens_per_item, static_cast<long long>(tokens_per_item) * (empty + 1) + prefix + kKeyTile - 1);
    if (r == row_tiles && row_tiles > 0) total += tiles_of(row_tiles - 1);
    return total;
  }
  FT_HD long long tiles_per_head() const { return row_tiles == 0 ? 0 : tiles_before(row_tiles); }
};

}  // namespace ftg
