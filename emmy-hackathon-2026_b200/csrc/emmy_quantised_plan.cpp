// emmy_quantised_plan.cpp -- cuts the attention over an 8-bit cache into work.
//
// A sequence whose query rows of a key head are few (few_rows) is bound by reading
// its keys, which a kernel of its own takes as they lie: its slices of keys are
// poured over the CTAs up to a common level, an item being cut where a CTA is full.
// The pieces go to the CTA's warps together or to each on its own (below).
// With more rows, which the tensor-core kernel takes, the keys are widened within it
// (middle), or read back to 16 bits once, in pages of 128 tokens, where many tiles of
// rows use them (many).  Little work goes to the first kernel whatever its rows.
#include "emmy_quantised.h"

#include <algorithm>
#include <cstdio>
#include <cstring>
#include <memory>
#include <new>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

using namespace emmy_quantised;

namespace {

// What a piece costs beside its slices, in slices of a warp (1.5 us where all warps of
// the GPU read): one that a CTA's warps share, for their waiting for one another and
// joining, and one of a warp.  Slices that are worth a shared piece or one of a warp;
// parts up to which an item is left to its warps (131,071 keys of one sequence: 53 us
// shared in 37 parts, 69 in 296; 8 sequences of 8,191: 36 us shared, 33 in 48 parts).
constexpr int kSharedCost = 5, kOwnCost = 2, kMinShared = 16, kMinOwn = 4, kMostParts = 64;
constexpr int kCtasAnSm = 2;
// 8-bit keys and values of sequences that are read back with others, though a kernel
// would take them as they are: 15 tokens (120 rows) over 4,110 keys of 4 heads of 64 took
// 46 us on 64 SMs before 138 us for seven sequences with more.
constexpr int64_t kSmallBytes = 32 << 20;
// Units x keys x blocks x head_dim^2 up to which more rows go to the kernel for few:
// heads of 128, one sequence of 8,192 keys and 8 heads: 32 rows 18 us against 23, 64 rows
// 26 and 30; of 32,768 keys: 32 rows (2^36) 35 and 41, 64 rows 60 and 54; 400 rows over 1,000 keys 21
// and 30; 8 sequences of 2,000 keys (2^38): 32 rows 25 and 23.  32 heads of 64, 2,000 keys:
// 64 rows 19 and 22.
constexpr int kFewBlock = 16;
constexpr double kIdle = 68719476736.0;      // 2^36
// Key tiles of a part where more than 32 rows share a tile: each part leaves 128 rows for
// the last to join.  1 sequence of 8,192 keys, 8 heads of 128: 256 rows 38 us, 44 with parts
// of 2, 41 of 16; 600 rows 81, 100 and 76; 16 of up to 8,192, 68 to 128 rows 88, 95, 87.
constexpr int kLeastPart = 8;

int fail(const char *fmt, long a = 0, long b = 0) {
  char buf[256];
  snprintf(buf, sizeof buf, fmt, a, b);
  return emmy_internal_fail(EMMY_EINVAL, buf);
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles of 8 query rows that the kernel for few rows computes, 1 or 2: more of them
// take a slice of keys longer, fewer read some keys twice.  Measured on 32 and 24
// sequences of up to 8,191 and 4,095 keys: 16 rows of 128 components take 1.17 of the
// time of 8, of 64 components 1.35.
int few_tiles(const emmy_paged_plan_args &a, const std::vector<uint8_t> &kind) {
  int64_t one = 0, two = 0;
  for (int s = 0; s < a.sequences; ++s) {
    const int64_t rows = int64_t(a.q_lens[s]) * (a.q_heads / a.kv_heads);
    if (kind[s]) continue;
    one += a.kv_lens[s] * div_up(rows, 8) * 100;
    two += a.kv_lens[s] * div_up(rows, 16) * (a.head_dim == 128 ? 117 : 135);
  }
  return one <= two ? 1 : 2;
}

void make(const emmy_paged_plan_args &a, emmy_quantised_plan_s &plan) {
  const int group = a.q_heads / a.kv_heads;
  // which kernels a sequence goes to
  enum { kFew, kMiddle, kMany };
  std::vector<uint8_t> kind(a.sequences);
  bool any[3] = {};
  for (int s = 0; s < a.sequences; ++s) {
    const int64_t rows = int64_t(a.q_lens[s]) * group;
    kind[s] = rows <= few_rows(a.head_dim) ? kFew : rows <= middle_rows(a.head_dim) ? kMiddle : kMany;
    plan.max_kv = std::max(plan.max_kv, a.kv_lens[s]);
  }
  // Work that would leave most of the GPU idle goes to the kernel for few rows, which cuts
  // it finest, in blocks of kFewBlock rows.  Its time grows with the keys times the blocks
  // that read them; the others' shrinks with the units that they have.
  auto keys_of = [&](int s) {
    return a.window ? std::min<int64_t>(a.kv_lens[s], int64_t(a.window) + a.q_lens[s]) : int64_t(a.kv_lens[s]);
  };
  for (const int least : {kMiddle, kMany}) {       // with the fewer rows alone only where there are no others
    int64_t units = 0, pieces = 0, read = 0, others = 0;
    for (int s = 0; s < a.sequences; ++s) {
      if (!a.q_lens[s] || kind[s] == kFew) continue;
      const int64_t rows = int64_t(a.q_lens[s]) * group, blocks = div_up(rows, kFewBlock);
      if (kind[s] > least || rows * group >= kMostRowsGroup) ++others;
      units += a.kv_heads;
      pieces += blocks * a.kv_heads;
      read += keys_of(s) * blocks * a.kv_heads;
    }
    if (others || pieces > int64_t(kCtasAnSm) * a.ctas) continue;
    if (double(units) * double(read) * (a.head_dim * a.head_dim) <= kIdle)
      for (int s = 0; s < a.sequences; ++s) kind[s] = kFew;
  }
  // Launches that would not fill the GPU one after the other are one: where some
  // sequences are read back, others of few bytes are too.
  int64_t bytes[3] = {}, small = 0;
  for (int s = 0; s < a.sequences; ++s)
    if (a.q_lens[s]) bytes[kind[s]] += keys_of(s) * a.kv_heads * a.head_dim * 2;
  for (const int k : {kMiddle, kFew})
    if (bytes[kMany] && bytes[k] && small + bytes[k] <= kSmallBytes) {
      small += bytes[k];
      for (int s = 0; s < a.sequences; ++s)
        if (kind[s] == k && a.q_lens[s]) kind[s] = kMany;
    }
  for (int s = 0; s < a.sequences; ++s) any[kind[s]] = true;
  plan.tiles = few_tiles(a, kind);
  const int keys = slice_keys(a.head_dim);
  const int at_once = 8 * plan.tiles;

  // the items of a sequence and a block of its rows, one for each key head
  struct Rows { int seq, row0, nslices; size_t first; bool own; };
  std::vector<Rows> blocks;
  std::vector<Piece> items;
  std::vector<Job> jobs;
  std::vector<int32_t> table;
  int64_t first = 0;
  for (int s = 0; s < a.sequences; ++s) {
    const int n = a.q_lens[s], len = a.kv_lens[s], pos0 = len - n;
    // keys that new tokens from..to-1 see between them
    auto lowest = [&](int from) { return a.window ? std::max(0, pos0 + from - a.window + 1) : 0; };
    auto highest = [&](int to) { return a.causal ? std::max(0, std::min(len, pos0 + to)) : len; };
    if (kind[s] == kFew) {
      for (int r = 0; r < n * group; r += at_once) {
        Piece p;
        memset(&p, 0, sizeof p);
        p.seq = s;
        p.tok0 = static_cast<int32_t>(first);
        p.row0 = r;
        p.rows = std::min(at_once, n * group - r);
        p.pos0 = pos0;
        p.kv_len = len;
        p.lo = lowest(r / group);
        p.hi = highest((r + p.rows - 1) / group + 1);
        p.nsplit = 1;
        if (p.hi > p.lo) {
          p.slice0 = p.lo / keys;
          p.nslices = (p.hi - 1) / keys + 1 - p.slice0;
          plan.reads = true;
        }
        blocks.push_back({s, r, p.nslices, items.size(), false});
        if (items.size() + a.kv_heads > (size_t(1) << 26)) throw 1;
        for (p.kvh = 0; p.kvh < a.kv_heads; ++p.kvh) items.push_back(p);
      }
    } else if (highest(n) > lowest(0)) {
      plan.reads = true;
      for (int b = lowest(0) / kBlock; kind[s] == kMany && b * kBlock < highest(n); ++b) {
        // (a token that no row sees is not used, but lies in a page that is)
        if (plan.workspace_pages >= (int64_t(1) << 26)) throw 1;
        jobs.push_back({s, b * kBlock, std::min(kBlock, len - b * kBlock), static_cast<int32_t>(plan.workspace_pages++)});
      }
    }
    first += n;
  }
  plan.tokens = first;

  // A CTA's warps either share a piece, or take a head each of some slices (`heads` of
  // them, and the slices in `ways` where there are more warps than heads): then nothing
  // waits for anything, and the heads of a token, which lie together, are read at about
  // the same time.  That is for work enough for all warps, and for sequences short
  // enough to be cut into few parts.
  const int warps = warps_of(plan.tiles), slots = kCtasAnSm * a.ctas;
  int heads = 1;
  for (int h = 2; h <= warps; ++h)
    if (warps % h == 0 && a.kv_heads % h == 0) heads = h;
  const int ways = warps / heads;
  int64_t total = 0;
  for (const Piece &p : items) total += p.nslices;
  const int64_t level0 = div_up(total, int64_t(slots) * warps);        // slices of a warp
  for (Rows &b : blocks) b.own = level0 >= 2 * kMinOwn && (b.nslices / (level0 * ways) + 2) * ways <= kMostParts;
  std::stable_partition(blocks.begin(), blocks.end(), [](const Rows &b) { return !b.own; });

  // the lowest level up to which the items fit on the CTAs
  struct Part { size_t item; int cta, warp, b, e; };      // warp -1: shared
  std::vector<Part> parts;
  auto pour = [&](int64_t level) {
    parts.clear();
    int c = 0;
    int64_t filled = 0;
    for (const Rows &rows : blocks)
      for (int h = 0; h < a.kv_heads; h += rows.own ? heads : 1) {
        const int per = rows.own ? ways : warps, cost = rows.own ? kOwnCost : kSharedCost;
        const int worth = rows.own ? kMinOwn * ways : kMinShared;
        int b = 0;
        do {
          const int rest = rows.nslices - b, least = std::min(worth, std::max(1, rest));
          while ((level - filled - cost) * per < least) {
            if (++c == slots) return false;
            filled = 0;
          }
          const int64_t room = (level - filled - cost) * per;
          // a rest too small to be a piece of its own goes along
          const int take = rest - room >= worth ? static_cast<int>(room) : rest;
          if (rows.own) {
            for (int k = 0; k < ways; ++k) {
              const int from = b + static_cast<int>(int64_t(take) * k / ways), to = b + static_cast<int>(int64_t(take) * (k + 1) / ways);
              if (to > from || (take == 0 && k == 0))
                for (int i = 0; i < heads; ++i) parts.push_back({rows.first + h + i, c, k * heads + i, from, to});
            }
          } else {
            parts.push_back({rows.first + h, c, -1, b, b + take});
          }
          filled += cost + div_up(take, per);
          b += take;
        } while (b < rows.nslices);
      }
    return true;
  };
  std::vector<std::vector<Piece>> dealt(slots * (warps + 1));
  std::vector<Joined> joined;
  if (!items.empty()) {
    int64_t low = 0, high = kSharedCost + kMinShared;
    while (!pour(high)) {
      low = high;
      high *= 2;
    }
    while (high - low > 1) {
      const int64_t mid = low + (high - low) / 2;
      (pour(mid) ? high : low) = mid;
    }
    pour(high);
    // the parts of an item in the order of their slices
    std::stable_sort(parts.begin(), parts.end(), [](const Part &x, const Part &y) { return x.item != y.item ? x.item < y.item : x.b < y.b; });
    for (size_t i = 0; i < parts.size();) {
      size_t e = i + 1;
      while (e < parts.size() && parts[e].item == parts[i].item) ++e;
      Piece p = items[parts[i].item];
      p.nsplit = static_cast<int32_t>(e - i);
      if (p.nsplit > 1) {
        if (plan.part_rows > (int64_t(1) << 30)) throw 1;
        p.part_row = static_cast<int32_t>(plan.part_rows);
        for (int r = 0; r < p.rows; ++r)
          joined.push_back({p.part_row + r, p.rows, p.nsplit, p.tok0 + (p.row0 + r) / group, p.kvh * group + (p.row0 + r) % group, {0, 0, 0}});
        plan.part_rows += int64_t(p.nsplit) * p.rows;
      }
      const int slice0 = p.slice0;
      for (size_t k = i; k < e; ++k) {
        p.slice0 = slice0 + parts[k].b;
        p.nslices = parts[k].e - parts[k].b;
        p.split = static_cast<int32_t>(k - i);
        dealt[parts[k].cta * (warps + 1) + parts[k].warp + 1].push_back(p);
      }
      i = e;
    }
  }
  // (CTAs are filled in their order: those with work come first, and the others are not launched)
  int used = 0;
  for (int c = 0; c < slots; ++c)
    for (int w = 0; w <= warps; ++w)
      if (!dealt[c * (warps + 1) + w].empty()) used = c + 1;
  size_t n_pieces = 0;
  for (const auto &d : dealt) n_pieces += d.size();

  auto plan_of = [&](int which) {
    std::vector<uint8_t> left_out(a.sequences);
    for (int s = 0; s < a.sequences; ++s) left_out[s] = kind[s] != which;
    emmy_paged_plan_t made = nullptr;
    if (any[which] && emmy_internal_paged_plan(&a, left_out.data(), which == kMiddle, kLeastPart, &made)) throw 2;
    return made;
  };
  plan.middle = plan_of(kMiddle);
  plan.many = plan_of(kMany);
  // (its kernel without the few rows' code, which costs the chunks 7 %: 174 us against 162)
  if (plan.many && plan.many->spread) plan.many->spread = false, plan.many->tiled = true;
  if (plan.many) {
    plan.table_width = static_cast<int32_t>(div_up(plan.many->max_kv, kBlock));
    table.assign(int64_t(a.sequences) * plan.table_width, 0);
    for (const Job &j : jobs) table[int64_t(j.seq) * plan.table_width + j.first / kBlock] = j.page;
    plan.n_jobs = static_cast<int32_t>(jobs.size());
  }

  Layout &at = plan.at;
  int64_t words = 4 + int64_t(used) * (warps + 1) + 1;
  auto place = [&](int64_t count, int64_t grid) {
    const int64_t begin = div_up(words, grid) * grid;
    words = begin + count;
    return begin;
  };
  const int64_t at_pieces = place(16 * int64_t(n_pieces), 16), at_joined = place(8 * int64_t(joined.size()), 8),
                at_middle = place(plan.middle ? int64_t(plan.middle->words.size()) : 0, 16),
                at_many = place(plan.many ? int64_t(plan.many->words.size()) : 0, 16),
                at_table = place(int64_t(table.size()), 4), at_jobs = place(4 * int64_t(jobs.size()), 4);
  if (words > (int64_t(1) << 30)) throw 1;
  at.ctas = used;
  at.pieces = static_cast<int>(at_pieces);
  at.joined = static_cast<int>(at_joined);
  plan.n_joined = static_cast<int32_t>(joined.size());
  at.middle = static_cast<int>(at_middle);
  at.many = static_cast<int>(at_many);
  at.table = static_cast<int>(at_table);
  at.jobs = static_cast<int>(at_jobs);
  plan.words.assign(words, 0);
  size_t k = 0;
  const int lists = used * (warps + 1);
  for (int i = 0; i < lists; ++i) {
    plan.words[4 + i] = static_cast<int32_t>(k);
    if (!dealt[i].empty()) memcpy(&plan.words[at.pieces + 16 * k], dealt[i].data(), dealt[i].size() * sizeof(Piece));
    k += dealt[i].size();
  }
  plan.words[4 + lists] = static_cast<int32_t>(k);
  plan.words[0] = used;
  plan.words[1] = warps;
  plan.words[2] = at.pieces;
  if (!joined.empty()) memcpy(&plan.words[at.joined], joined.data(), sizeof(Joined) * joined.size());
  if (plan.middle) memcpy(&plan.words[at.middle], plan.middle->words.data(), 4 * plan.middle->words.size());
  if (plan.many) memcpy(&plan.words[at.many], plan.many->words.data(), 4 * plan.many->words.size());
  if (!table.empty()) memcpy(&plan.words[at.table], table.data(), 4 * table.size());
  if (!jobs.empty()) memcpy(&plan.words[at.jobs], jobs.data(), sizeof(Job) * jobs.size());
}

}  // namespace

extern "C" EMMY_API int emmy_quantised_plan_make(const emmy_paged_plan_args *a, emmy_quantised_plan_t *out) {
  if (!a || !out || a->sequences < 0 || (a->sequences && (!a->q_lens || !a->kv_lens)))
    return fail("emmy_quantised_plan_make: bad argument");
  *out = nullptr;
  if (a->kv_heads < 1 || a->q_heads < 1 || a->q_heads % a->kv_heads || a->q_heads / a->kv_heads > 128)
    return fail("emmy_quantised_plan_make: %ld query heads for %ld key heads (1 to 128 times as many)", a->q_heads, a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128) return fail("emmy_quantised_plan_make: head_dim %ld (64 or 128)", a->head_dim);
  if (a->window < 0 || (a->window && !a->causal))
    return fail("emmy_quantised_plan_make: window %ld (a window is causal)", a->window);
  if (a->ctas < 1 || a->ctas > 65536) return fail("emmy_quantised_plan_make: %ld CTAs", a->ctas);
  int64_t tokens = 0;
  int32_t longest = 0;
  for (int s = 0; s < a->sequences; ++s) {
    if (a->q_lens[s] < 0 || a->kv_lens[s] < 0 || a->q_lens[s] > (1 << 30) || a->kv_lens[s] > (1 << 30))
      return fail("emmy_quantised_plan_make: sequence %ld has a length outside 0..2^30", s);
    tokens += a->q_lens[s];
    longest = std::max(longest, a->kv_lens[s]);
  }
  emmy_paged_plan_args args = *a;
  if (args.window >= longest) args.window = 0;      // (hides no key)
  if (tokens * a->q_heads > (int64_t(1) << 30)) return fail("emmy_quantised_plan_make: too many tokens");
  try {
    std::unique_ptr<emmy_quantised_plan_s> plan(new emmy_quantised_plan_s);
    plan->sequences = a->sequences;
    plan->q_heads = a->q_heads;
    plan->kv_heads = a->kv_heads;
    plan->head_dim = a->head_dim;
    plan->causal = a->causal != 0;
    plan->window = args.window;
    make(args, *plan);
    *out = plan.release();
    return 0;
  } catch (const std::bad_alloc &) {
    return emmy_internal_fail(EMMY_ENOMEM, "emmy_quantised_plan_make: out of host memory");
  } catch (int) {
    return emmy_internal_fail(EMMY_EINVAL, "emmy_quantised_plan_make: too much work for one plan");
  } catch (...) {
    return emmy_internal_fail(EMMY_EINVAL, "emmy_quantised_plan_make: failed");
  }
}

extern "C" EMMY_API int emmy_quantised_plan_data(emmy_quantised_plan_t plan, const int32_t **words, size_t *n_words, size_t *scratch) {
  if (!plan || !words || !n_words || !scratch) return fail("emmy_quantised_plan_data: bad argument");
  *words = plan->words.data();
  *n_words = plan->words.size();
  *scratch = emmy_quantised::scratch_of(*plan).end;
  return 0;
}

extern "C" EMMY_API void emmy_quantised_plan_free(emmy_quantised_plan_t plan) { delete plan; }
