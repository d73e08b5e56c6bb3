// emmy_quantised.h -- what the plan (host) and the kernels of attention over an
// 8-bit cache share.
#pragma once
#include "emmy_paged.h"

#include <vector>

namespace emmy_quantised {

constexpr int slice_keys(int head_dim) { return 2048 / head_dim; }      // that a warp takes at once: 2 KiB of 8-bit keys
// Query rows of a sequence and key head up to which they are few, and up to which the
// tensor-core kernel widens its keys itself (128 rows at a time) instead of reading them
// back.  32 sequences of up to 8,191 keys, 8 heads of 128: 17 rows 128 us widened, 136 as
// few; 384 rows 431 widened, 504 read back; 512 rows 565 and 503.  24 of up to 4,095, 32
// heads of 64: 24 rows 130 us as few, 140 widened; 32 rows 138 and 135; 128 rows 200
// widened, 278 read back; 160 rows 374 and 328.
constexpr int few_rows(int head_dim) { return head_dim == 128 ? 16 : 24; }
constexpr int middle_rows(int head_dim) { return head_dim == 128 ? 384 : 128; }
// The kernel for few rows divides a sequence's row r by G as r * ceil(2^16 / G) >> 16, which
// is too large by less than r G / 2^16 of 1 / G: right for r G under 2^16, and in 32 bits
// for r / G under 2^15.
constexpr int64_t kMostRowsGroup = 1 << 15;
constexpr int kBlock = 128;         // tokens of a page of the workspace, which keys are read back to

// Warps of a CTA whose pieces have one or two tiles of 8 query rows: as many as the
// registers of their sums allow twice an SM (128 or 168 a thread).
constexpr int warps_of(int tiles) { return tiles == 1 ? 8 : 6; }

// A piece of work: up to 8 or 16 query rows of one sequence and key head (row r is
// new token (row0 + r) / G of the sequence, query head (row0 + r) % G of the group)
// against some of the key slices that they see between them.  The warps of a CTA share
// its `shared` pieces, slice by slice in turn, and have others of their own after
// them.  `nsplit` pieces share an item: each leaves a partial result in its rows of the
// scratch, which a kernel of its own joins.
struct Piece {
  int32_t seq, kvh;
  int32_t tok0;             // the sequence's first row of q
  int32_t row0, rows;
  int32_t pos0;             // position of the sequence's first new token (negative: sees no key)
  int32_t lo, hi;           // keys that the item's rows see between them
  int32_t kv_len;
  int32_t slice0, nslices;
  int32_t split, nsplit;
  int32_t part_row;         // first scratch row of the item
  int32_t pad[2];
};
static_assert(sizeof(Piece) == 64, "pieces are read as 64-byte records");

// A row of an item of several parts: where the first part's is, how many rows one
// part is from the next, and where the result goes.
struct Joined { int32_t part_row, step, nsplit, token, head, pad[3]; };
static_assert(sizeof(Joined) == 32, "rows are read as two 16-byte records");

struct Job { int32_t seq, first, count, page; };      // read back: tokens first..first+count of a sequence, to a page
static_assert(sizeof(Job) == 16, "jobs are read as 16-byte records");

// The plan's words on the device, by their offsets: CTAs, warps of one, offset of the
// pieces, the status; from 4 on where the pieces of each CTA begin that its warps share
// and then those of each warp (ctas x (warps + 1) + 1); pieces, rows to join, the words
// of the plans of the sequences with more rows, middle and many (emmy_paged.h), the page
// table [sequences][width] of the latter in the workspace, and the jobs that fill it.  The kernels write the
// status (that of every kernel of a call: where one gave up none does any more) and what the other plans have of their own.
struct Layout {
  static constexpr int status = 3;
  int ctas = 0, pieces = 0, joined = 0, middle = 0, many = 0, table = 0, jobs = 0;
};

}  // namespace emmy_quantised

struct emmy_quantised_plan_s {
  std::vector<int32_t> words;
  emmy_quantised::Layout at;
  emmy_paged_plan_s *middle = nullptr, *many = nullptr;       // of the sequences with more rows; null: none
  int64_t tokens = 0, part_rows = 0, workspace_pages = 0;
  int32_t sequences = 0, q_heads = 0, kv_heads = 0, head_dim = 0, causal = 0, window = 0, max_kv = 0;
  int32_t tiles = 1;                         // tiles of 8 rows that a piece may have: 1 or 2
  int32_t table_width = 0, n_jobs = 0, n_joined = 0;
  bool reads = false;                        // some row sees a key
  ~emmy_quantised_plan_s() {
    delete middle;
    delete many;
  }
};

namespace emmy_quantised {

// The scratch by its offsets, multiples of 128 bytes: partial rows of head_dim floats
// with (base, sum, c) of each; those of the other plans; 16-bit keys and values read back.
struct Scratch { size_t middle, many, workspace, end; };
inline Scratch scratch_of(const emmy_quantised_plan_s &plan) {
  auto whole = [](size_t bytes) { return (bytes + 127) / 128 * 128; };
  auto others = [&](const emmy_paged_plan_s *p) { return p ? whole(size_t(p->part_rows) * (plan.head_dim + 2) * sizeof(float)) : 0; };
  Scratch at;
  at.middle = whole(size_t(plan.part_rows) * (plan.head_dim + 4) * sizeof(float));
  at.many = at.middle + others(plan.middle);
  at.workspace = at.many + others(plan.many);
  at.end = at.workspace + size_t(plan.workspace_pages) * kBlock * plan.kv_heads * plan.head_dim * 2 * 2;
  return at;
}

}  // namespace emmy_quantised

// emmy_paged_plan.cpp: a plan without the sequences that left_out marks, whose rows it
// leaves alone; `narrow`: without wide units; least_part: key tiles of a part of a narrow unit
// of more than 32 rows
int emmy_internal_paged_plan(const emmy_paged_plan_args *a, const uint8_t *left_out, bool narrow, int least_part, emmy_paged_plan_t *out);
// emmy_paged_attention.cu: as a part of a plan whose status is at batch_status; bits8: over a cache of 8-bit floats
int emmy_internal_paged_attention(emmy_paged_plan_t plan, const emmy_paged_attention_args *a, bool bits8, uint64_t exponents, uint64_t batch_status,
                                  void *stream);
