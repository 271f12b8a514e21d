// How the attention over packed prompts and over the cache is cut into equal shares: plain integer arithmetic, the same
// on the device and on the host (where it is tested).
//
// A sequence of n queries and some keys makes, for each key head, ceil(n / tokens_per_item) row tiles; a row tile works
// through the 128-key tiles that any of its rows may see.  To begin and end a row tile costs about as much as item_cost
// key tiles, so a row tile of T key tiles is T + item_cost units of work, the first item_cost of them without a key tile.
// The units of all row tiles, heads and sequences are numbered in a row, and CTA c takes [c * share, (c + 1) * share); a
// row tile whose first key tile lies in a share's front belongs to that share from its beginning.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FT_HD __host__ __device__ __forceinline__
#else
#define FT_HD inline
#endif

namespace ftg {

constexpr int kKeyTile = 128;

// All units of a call are numbered in 31 bits (more are refused: at a microsecond each they would take seconds on every SM
// of the device).

// sum over i in [0, n) of floor((a i + b) / 128) for a, b >= 0.  The steps repeat every 128 / gcd(a, 128) terms with an
// increment of a / gcd(a, 128): one period is added up term by term (at most 128 of them; at most 4 for the usual head
// groups), the rest follows.
FT_HD int floor_sum(int n, int a, int b) {
  if (n <= 0) return 0;
  int shift = 0;  // period = 2^shift
  while (((a << shift) & (kKeyTile - 1)) != 0) ++shift;
  const int period = 1 << shift, step = (a << shift) / kKeyTile, periods = n >> shift, rest = n & (period - 1);
  int one = 0, head = 0;  // a whole period, and its first `rest` terms
  int at = b;
#pragma unroll 1
  for (int i = 0; i < period; ++i, at += a) {
    if (i == rest) head = one;
    one += at / kKeyTile;
  }
  return periods * one + step * period * static_cast<int>(static_cast<long long>(periods) * (periods - 1) / 2) + head + rest * periods * step;
}

struct SequenceTiles {
  int queries, keys;    // keys: how many may be read
  int prefix;           // key tokens in front of the first query's own (negative: the first queries see nothing)
  int row_tiles;        // per key head
  int tokens_per_item;
  int item_cost;
  bool chain;           // query t sees keys [0, prefix + t]; otherwise row tiles count all keys
  bool ramp;            // row tiles are numbered with their own key limit; otherwise with all keys

  FT_HD static SequenceTiles make(int queries, int keys, int full_keys, int tokens_per_item, int item_cost, bool chain) {
    SequenceTiles s;
    s.queries = queries;
    s.keys = keys;
    s.prefix = full_keys - queries;
    s.tokens_per_item = tokens_per_item;
    s.item_cost = item_cost;
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
    if (!ramp) return tiles(keys) + item_cost;
    const long long end = static_cast<long long>(r + 1) * tokens_per_item;
    return tiles(limit(end < queries ? static_cast<int>(end) : queries)) + item_cost;
  }
  // units of the row tiles in front of r, r in [0, row_tiles]
  FT_HD int units_before(int r) const {
    if (!ramp) return r * (tiles(keys) + item_cost);
    const int inner = r < row_tiles ? r : row_tiles - 1;  // the last row tile ends with the queries, not on the line
    int empty = 0;                                        // row tiles that see nothing
    if (prefix < 0) {
      empty = -prefix / tokens_per_item;
      empty = empty > inner ? inner : empty;
    }
    int total = inner * item_cost + empty + floor_sum(inner - empty, tokens_per_item, tokens_per_item * (empty + 1) + prefix + kKeyTile - 1);
    if (r == row_tiles && row_tiles > 0) total += units_of(row_tiles - 1);
    return total;
  }
  // at least the units of a key head, in 64 bits: every row tile with all keys
  FT_HD long long most_units_per_head() const { return static_cast<long long>(row_tiles) * (tiles(keys) + item_cost); }
  FT_HD int units_per_head() const { return row_tiles == 0 ? 0 : units_before(row_tiles); }
};

}  // namespace ftg
