// emmy_paged.h -- what the paged attention's plan (host) and kernel share.
#pragma once
#include "../../include/emmy_b200.h"

#include <vector>

namespace emmy_paged {

constexpr int kTile = 128;          // keys of a tile, and rows of a tile of queries

// A unit: up to two query tiles of one sequence and key head (tile t's row r is
// new token t * tokens_per_tile + r / G of the unit, query head r % G of the
// group) against `ntiles` key tiles.  More than one tile of queries is a `wide`
// unit.  An item is the same queries against all their keys; `nsplit` units
// share one, each leaving a partial result in its rows of the scratch.  A CTA's
// wide units come before its others: the kernel relies on that (a unit of few rows
// joins its results where the second tile of queries of a wide unit would lie).
struct Unit {
  int32_t seq, kvh;
  int32_t tok0, ntok;       // first row of q, new tokens
  int32_t pos0;             // position of the first token (negative: sees no key)
  int32_t tile0, ntiles;    // key tiles of this unit
  int32_t lo, hi;           // keys that the item's tokens see between them
  int32_t kv_len;
  int32_t wide;
  int32_t item, split, nsplit;   // item: index of its arrival counters
  int32_t part_row;         // first scratch row of the item
  int32_t pad;
};
static_assert(sizeof(Unit) == 64, "units are read as 64-byte records, four fields at a time");

// Words on the device: status, ctas, offsets of the counters and of the units,
// cta_first[ctas + 1], counters[2 * items], then the units at the next multiple
// of 16 words.  The kernel writes the status and the counters only, and leaves
// the counters at 0.
struct Layout {
  int ctas = 0, counters = 0, units = 0;     // word offsets of the last two
  int n_units = 0;
};

// The few rows of a unit are spread over a stream's warps (ntiles of the unit or
// of any part of its item).
#ifdef __CUDACC__
__host__ __device__
#endif
inline bool is_spread(int wide, int ntiles, int ntok, int group) { return !wide && ntiles && ntok * group <= 32; }

}  // namespace emmy_paged

struct emmy_paged_plan_s {
  std::vector<int32_t> words;
  emmy_paged::Layout at;
  int64_t tokens = 0;
  int64_t part_rows = 0;
  bool tiled = false, spread = false;      // some unit has whole query tiles, or rows for one warp
  bool narrow = false;                     // made without wide units
  int32_t sequences = 0, q_heads = 0, kv_heads = 0, head_dim = 0, causal = 0, window = 0, max_kv = 0;
};
