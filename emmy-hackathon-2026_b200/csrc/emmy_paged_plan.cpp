// emmy_paged_plan.cpp -- cuts the paged attention's work into units and deals
// them to the CTAs.
//
// Wide units (two tiles of queries) are bound by the tensor cores and leave a
// large partial result when cut, so they stay whole unless there are too few to
// fill the GPU, and go to the CTA with the least work so far in an order in which
// CTAs that run at the same time share a head's keys in L2.  Units of one query
// tile are bound by reading their keys and leave a small partial result, so
// they are poured over the CTAs up to a common level, cut where a CTA is full.
#include "emmy_paged.h"

#include <algorithm>
#include <cstdio>
#include <cstring>
#include <new>
#include <queue>

int emmy_internal_fail(int code, const char *msg);   // emmy_runtime.cpp

using emmy_paged::kTile;
using emmy_paged::Unit;

namespace {

// What work costs, in quarters of the time of a key tile of one query tile (0.73
// us with 64 components, 1.37 with 128, bound by memory): measured on calls of
// 148 equal units of 64 to 256 tiles, and of 8 x 148 units of 8.  A wide tile is
// bound by its softmax, the same for either; a unit's end drains and joins its
// streams; a part of a cut wide unit goes through the scratch besides.
struct Cost { int64_t narrow_tile, narrow_unit, wide_tile, wide_unit, wide_part; };
constexpr Cost kCost64 = {4, 18, 7, 25, 22}, kCost128 = {4, 6, 4, 16, 12};
constexpr int kMinNarrow = 2;    // tiles: the two streams of a CTA take one each
constexpr int kMinWide = 4;      // tiles: under this a part is all overhead

int fail(const char *fmt, long a = 0, long b = 0) {
  char buf[256];
  snprintf(buf, sizeof buf, fmt, a, b);
  return emmy_internal_fail(EMMY_EINVAL, buf);
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

void make(const emmy_paged_plan_args &a, emmy_paged_plan_s &plan) {
  const int group = a.q_heads / a.kv_heads, per_tile = kTile / group;
  const Cost cost = a.head_dim == 64 ? kCost64 : kCost128;
  std::vector<Unit> wide, narrow;     // one unit an item, to be cut below
  int64_t first = 0;
  for (int s = 0; s < a.sequences; ++s) {
    const int n = a.q_lens[s], len = a.kv_lens[s];
    plan.max_kv = std::max(plan.max_kv, len);
    const int blocks = static_cast<int>(div_up(n, 2 * per_tile));
    for (int h = 0; h < a.kv_heads; ++h)
      for (int b = blocks - 1; b >= 0; --b) {
        Unit u;
        memset(&u, 0, sizeof u);
        const int t0 = b * 2 * per_tile;
        u.seq = s;
        u.kvh = h;
        u.tok0 = static_cast<int32_t>(first + t0);
        u.ntok = std::min(2 * per_tile, n - t0);
        u.pos0 = len - n + t0;
        u.kv_len = len;
        u.hi = a.causal ? std::min(len, u.pos0 + u.ntok) : len;
        u.lo = a.window ? std::max(0, u.pos0 - a.window + 1) : 0;
        u.wide = u.ntok > per_tile;
        u.nsplit = 1;
        if (u.hi > u.lo) {
          u.tile0 = u.lo / kTile;
          u.ntiles = (u.hi - 1) / kTile + 1 - u.tile0;
        }
        const bool spread = emmy_paged::is_spread(u.wide, u.ntiles, u.ntok, group);
        plan.spread = plan.spread || spread;
        plan.tiled = plan.tiled || (u.ntiles && !spread);
        (u.wide ? wide : narrow).push_back(u);
      }
    first += n;
  }
  plan.tokens = first;

  std::vector<std::vector<Unit>> dealt(a.ctas);
  std::vector<int64_t> load(a.ctas, 0);
  int items = 0;
  auto split_item = [&](const Unit &u, int nsplit) {     // rows of the scratch and counters
    Unit v = u;
    v.nsplit = nsplit;
    v.item = items++;
    v.part_row = static_cast<int32_t>(plan.part_rows);
    plan.part_rows += int64_t(nsplit) * u.ntok * group;
    return v;
  };

  // Wide units go out by head while they are long, so that CTAs share keys, and
  // then the short ones, longest first, to even out the ends.  The last units
  // may be cut by keys: of a few ways to cut, the one that ends first is taken.
  int longest = 0;
  for (const Unit &u : wide) longest = std::max(longest, u.ntiles);
  std::stable_sort(wide.begin(), wide.end(), [&](const Unit &x, const Unit &y) {
    const int kx = x.ntiles * 2 > longest ? longest + 1 : x.ntiles, ky = y.ntiles * 2 > longest ? longest + 1 : y.ntiles;
    return kx > ky;
  });
  struct Cut { size_t whole; int pieces; };       // units left whole, pieces of the others
  auto pieces_of = [&](const Cut &cut, size_t i) {
    return i < cut.whole ? 1 : std::max(1, std::min(cut.pieces, wide[i].ntiles / kMinWide));
  };
  auto part = [](const Unit &u, int k, int n) { return static_cast<int>(int64_t(u.ntiles) * k / n); };
  typedef std::pair<int64_t, int> Slot;
  auto deal = [&](const Cut &cut, bool keep) {    // greedy; the time that it ends
    std::vector<Slot> heap;
    for (int c = 0; c < a.ctas; ++c) heap.push_back({0, c});
    std::priority_queue<Slot, std::vector<Slot>, std::greater<Slot>> least(std::greater<Slot>(), std::move(heap));
    int64_t end = 0;
    for (size_t i = 0; i < wide.size(); ++i) {
      const int n = pieces_of(cut, i);
      Unit v = keep && n > 1 ? split_item(wide[i], n) : wide[i];
      for (int k = 0; k < n; ++k) {
        const int b = part(wide[i], k, n), e = part(wide[i], k + 1, n);
        Slot s = least.top();
        least.pop();
        s.first += cost.wide_unit + cost.wide_tile * (e - b) + (n > 1 ? cost.wide_part : 0);
        end = std::max(end, s.first);
        least.push(s);
        if (!keep) continue;
        v.tile0 = wide[i].tile0 + b;
        v.ntiles = e - b;
        v.split = k;
        dealt[s.second].push_back(v);
        load[s.second] = s.first;
      }
    }
    return end;
  };
  if (!wide.empty()) {
    Cut best = {wide.size(), 1};
    int64_t end = deal(best, false);
    // cutting costs the parts' way through the scratch: it has to gain 3 %
    int64_t total = 0;
    for (const Unit &u : wide) total += cost.wide_unit + cost.wide_tile * u.ntiles;
    const bool even = end * a.ctas * 100 <= total * 103;
    const size_t ctas = a.ctas, all = wide.size();
    for (const size_t last : {all % ctas, ctas, ctas + all % ctas, 2 * ctas})
      for (int n = 2; n <= 16 && !even; n *= 2) {
        const Cut cut = {all - std::min(all, last), n};
        const int64_t e = deal(cut, false);
        if (e * 103 < end * 100) {
          end = e;
          best = cut;
        }
      }
    deal(best, true);
  }

  // the lowest level up to which the narrow units fit on the CTAs
  struct Piece { int unit, cta, b, e; };
  std::vector<Piece> pieces;
  auto pour = [&](int64_t level) {
    pieces.clear();
    int c = 0;
    int64_t filled = load[0];
    for (size_t i = 0; i < narrow.size(); ++i) {
      int b = 0;
      do {
        const int rest = narrow[i].ntiles - b, least_take = std::min(kMinNarrow, std::max(1, rest));
        int64_t room = (level - filled - cost.narrow_unit) / cost.narrow_tile;
        while (room < least_take) {
          if (++c == a.ctas) return false;
          filled = load[c];
          room = (level - filled - cost.narrow_unit) / cost.narrow_tile;
        }
        // a rest too small to be a piece of its own goes along
        const int take = rest - room >= kMinNarrow ? static_cast<int>(room) : rest;
        pieces.push_back({static_cast<int>(i), c, b, b + take});
        filled += cost.narrow_unit + cost.narrow_tile * take;
        b += take;
      } while (b < narrow[i].ntiles);
    }
    return true;
  };
  if (!narrow.empty()) {
    int64_t high = cost.narrow_unit + cost.narrow_tile * kMinNarrow;
    for (const int64_t l : load) high = std::max(high, l);
    int64_t low = high;             // no CTA may stay under the level of the smallest piece
    for (const int64_t l : load) low = std::min(low, l);
    low = std::max(low, cost.narrow_unit + cost.narrow_tile * kMinNarrow - 1);
    while (!pour(high)) {
      low = high;
      high *= 2;
    }
    while (high - low > 1) {
      const int64_t mid = low + (high - low) / 2;
      (pour(mid) ? high : low) = mid;
    }
    pour(high);
    for (size_t i = 0; i < pieces.size();) {
      const Unit &u = narrow[pieces[i].unit];
      size_t e = i + 1;
      while (e < pieces.size() && pieces[e].unit == pieces[i].unit) ++e;
      Unit v = e - i > 1 ? split_item(u, static_cast<int>(e - i)) : u;
      for (size_t k = i; k < e; ++k) {
        v.tile0 = u.tile0 + pieces[k].b;
        v.ntiles = pieces[k].e - pieces[k].b;
        v.split = static_cast<int32_t>(k - i);
        dealt[pieces[k].cta].push_back(v);
      }
      i = e;
    }
  }

  // CTAs with work come first; the others are not launched
  std::stable_partition(dealt.begin(), dealt.end(), [](const std::vector<Unit> &d) { return !d.empty(); });
  int used = 0;
  while (used < a.ctas && !dealt[used].empty()) ++used;
  size_t n = 0;
  for (const auto &d : dealt) n += d.size();
  emmy_paged::Layout &at = plan.at;
  at.ctas = used;
  at.n_units = static_cast<int>(n);
  at.counters = 4 + used + 1;
  at.units = static_cast<int>(div_up(at.counters + 2 * items, 16) * 16);
  plan.words.assign(at.units + 16 * n, 0);
  plan.words[1] = used;
  plan.words[2] = at.counters;
  plan.words[3] = at.units;
  size_t k = 0;
  for (int i = 0; i < used; ++i) {
    plan.words[4 + i] = static_cast<int32_t>(k);
    memcpy(&plan.words[at.units + 16 * k], dealt[i].data(), dealt[i].size() * sizeof(Unit));
    k += dealt[i].size();
  }
  plan.words[4 + used] = static_cast<int32_t>(n);
}

}  // namespace

extern "C" EMMY_API int emmy_paged_plan_make(const emmy_paged_plan_args *a, emmy_paged_plan_t *out) {
  if (!a || !out || a->sequences < 0 || (a->sequences && (!a->q_lens || !a->kv_lens)))
    return fail("emmy_paged_plan_make: bad argument");
  *out = nullptr;
  if (a->kv_heads < 1 || a->q_heads < 1 || a->q_heads % a->kv_heads || a->q_heads / a->kv_heads > kTile)
    return fail("emmy_paged_plan_make: %ld query heads for %ld key heads (1 to 128 times as many)", a->q_heads, a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128) return fail("emmy_paged_plan_make: head_dim %ld (64 or 128)", a->head_dim);
  if (a->window < 0 || (a->window && !a->causal))
    return fail("emmy_paged_plan_make: window %ld (a window is causal)", a->window);
  if (a->ctas < 1 || a->ctas > 65536) return fail("emmy_paged_plan_make: %ld CTAs", a->ctas);
  int64_t tokens = 0;
  int32_t longest = 0;
  for (int s = 0; s < a->sequences; ++s) {
    if (a->q_lens[s] < 0 || a->kv_lens[s] < 0 || a->q_lens[s] > (1 << 30) || a->kv_lens[s] > (1 << 30))
      return fail("emmy_paged_plan_make: sequence %ld has a length outside 0..2^30", s);
    tokens += a->q_lens[s];
    longest = std::max(longest, a->kv_lens[s]);
  }
  // A window that hides no key is none; others, and the positions that they are taken
  // from, down to -2^30, are small enough for 32 bits here and in the kernel.
  emmy_paged_plan_args args = *a;
  if (args.window >= longest) args.window = 0;
  if (tokens * a->q_heads > (int64_t(1) << 30)) return fail("emmy_paged_plan_make: too many tokens");
  try {
    emmy_paged_plan_s *plan = new emmy_paged_plan_s;
    plan->sequences = a->sequences;
    plan->q_heads = a->q_heads;
    plan->kv_heads = a->kv_heads;
    plan->head_dim = a->head_dim;
    plan->causal = a->causal != 0;
    plan->window = args.window;
    try {
      make(args, *plan);
    } catch (...) {
      delete plan;
      throw;
    }
    if (plan->part_rows > (int64_t(1) << 31) - 1) {
      delete plan;
      return fail("emmy_paged_plan_make: too many partial rows");
    }
    *out = plan;
    return 0;
  } catch (const std::bad_alloc &) {
    return emmy_internal_fail(EMMY_ENOMEM, "emmy_paged_plan_make: out of host memory");
  } catch (...) {
    return emmy_internal_fail(EMMY_EINVAL, "emmy_paged_plan_make: failed");
  }
}

extern "C" EMMY_API int emmy_paged_plan_data(emmy_paged_plan_t plan, const int32_t **words, size_t *n_words,
                                             size_t *scratch) {
  if (!plan || !words || !n_words || !scratch) return fail("emmy_paged_plan_data: bad argument");
  *words = plan->words.data();
  *n_words = plan->words.size();
  // partial rows of head_dim floats, then (exponent base, sum) of each
  *scratch = size_t(plan->part_rows) * (plan->head_dim + 2) * sizeof(float);
  return 0;
}

extern "C" EMMY_API void emmy_paged_plan_free(emmy_paged_plan_t plan) { delete plan; }
