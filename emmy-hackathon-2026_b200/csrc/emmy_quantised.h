// emmy_quantised.h -- what the plan (host) and the kernels of attention over an
// 8-bit cache share.
#pragma once
#include "emmy_paged.h"

#include <vector>

namespace emmy_quantised {

constexpr int kSlice = 16;          // keys that a warp takes at once
constexpr int kFewRows = 128;       // query rows of a sequence and key head up to which they are few
constexpr int kBlock = 128;         // tokens of a page of the workspace, which the others' keys are read back to

// A piece of work of one CTA: up to 8 or 32 query rows of one sequence and key head
// (row r is new token (row0 + r) / G of the sequence, query head (row0 + r) % G of
// the group) against some of the key slices that they see between them.  `nsplit`
// pieces share an item: each leaves a partial result in its rows of the scratch, and
// the last to arrive joins them.
struct Piece {
  int32_t seq, kvh;
  int32_t tok0;             // the sequence's first row of q
  int32_t row0, rows;
  int32_t pos0;             // position of the sequence's first new token (negative: sees no key)
  int32_t lo, hi;           // keys that the item's rows see between them
  int32_t kv_len;
  int32_t slice0, nslices;
  int32_t item, split, nsplit;   // item: its arrival counter
  int32_t part_row;         // first scratch row of the item
  int32_t pad;
};
static_assert(sizeof(Piece) == 64, "pieces are read as 64-byte records");

struct Job { int32_t seq, first, count, page; };      // read back: tokens first..first+count of a sequence, to a page
static_assert(sizeof(Job) == 16, "jobs are read as 16-byte records");

// The plan's words on the device, by their offsets: cta_first[ctas + 1], the items'
// counters, pieces, the words of the plan of the others (emmy_paged.h), their page
// table [sequences][width] in the workspace, and the jobs that fill it.
struct Layout {
  int ctas = 0, counters = 0, pieces = 0, others = 0, table = 0, jobs = 0;
};

}  // namespace emmy_quantised

struct emmy_quantised_plan_s {
  std::vector<int32_t> words;
  emmy_quantised::Layout at;
  emmy_paged_plan_s *others = nullptr;       // of the sequences with many rows; null: none
  int64_t tokens = 0, part_rows = 0, workspace_pages = 0;
  int32_t sequences = 0, q_heads = 0, kv_heads = 0, head_dim = 0, causal = 0, window = 0, max_kv = 0;
  int32_t tiles = 1;                         // tiles of 8 rows that a piece may have: 1 or 4
  int32_t table_width = 0, n_jobs = 0;
  bool reads = false;                        // some row sees a key
  ~emmy_quantised_plan_s() { delete others; }
};

// emmy_paged_plan.cpp: a plan without the sequences that left_out marks, whose rows it leaves alone
int emmy_internal_paged_plan(const emmy_paged_plan_args *a, const uint8_t *left_out, emmy_paged_plan_t *out);
