// How attention over shared prefixes is cut into units of work (host code, no CUDA).
#pragma once
#include <algorithm>

// Kernels, by the query rows of a unit: a warp for up to 8, a CTA for up to 64, a CTA with tcgen05 products for up to 256; a CTA of
// multiply-adds for 16 in 32-bit formats.
enum : int { AP_ROWS = 0, AP_TILES = 1, AP_TC = 2, AP_PLAIN = 3 };

struct PrefixPart {
  int kernel;               // AP_*
  int tile;                 // query rows of a unit
  int tiles;                // of a group (an item) and key head
  int splits;               // ranges that the cached rows are cut into
  long long units;
};

struct PrefixPlan {
  PrefixPart shared, own;
  int together;             // both parts in one launch
  int parts;                // of a result
};

// `rows` query rows at each of `heads` (groups or items) x n_kv; `tc`: tcgen05 may be used.
inline PrefixPart prefix_part(long long heads, long long rows, int n_kv, bool wide, bool tc) {
  PrefixPart p{};
  p.kernel = wide ? AP_PLAIN : rows <= 8 ? AP_ROWS : rows <= 64 || !tc ? AP_TILES : AP_TC;
  p.tile = p.kernel == AP_PLAIN ? 16 : p.kernel == AP_ROWS ? 8 : p.kernel == AP_TC ? 256 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  p.tiles = (int)((rows + p.tile - 1) / p.tile);
  p.units = heads * n_kv * p.tiles;
  return p;
}
inline int prefix_cut(long long rows, long long chunk, long long most) {
  return (int)std::min(most, std::max(1LL, (rows + chunk - 1) / chunk));
}
// What runs at once is given about equal shares of `total` cached rows; four units each where they are long, so that lengths that
// differ even out.
inline long long prefix_chunk(long long total, long long at_once, long long least) {
  const long long each = total / at_once;
  return each < 4 * least ? std::max(least, each) : std::max(4 * least, each / 4);
}

// max_group items of `rep` heads share a group's rows.
inline PrefixPlan prefix_plan(long long n_groups, long long max_group, long long max_prefix, long long n_items, long long max_own, int n_kv,
                              int rep, bool wide, bool tc, int sms) {
  PrefixPlan p{};
  p.shared = prefix_part(n_groups, n_groups > 0 ? max_group * rep : 0, n_kv, wide, tc);
  p.own = prefix_part(n_items, max_own > 0 ? rep : 0, n_kv, wide, false);
  const bool any1 = n_groups > 0, any2 = max_own > 0;
  p.together = any1 && any2 && p.shared.kernel == p.own.kernel;
  const long long total1 = p.shared.units * max_prefix, total2 = p.own.units * max_own;
  const auto at_once = [&](int kernel) { return (long long)sms * (kernel == AP_ROWS ? 12 : 4); };
  const auto least = [](int kernel) { return kernel == AP_ROWS ? 64LL : 128LL; };
  if (any2) p.own.splits = prefix_cut(max_own, prefix_chunk(total2 + (p.together ? total1 : 0), at_once(p.own.kernel), least(p.own.kernel)), 32);
  if (any1 && p.shared.kernel != AP_TC) {
    p.shared.splits = prefix_cut(max_prefix, prefix_chunk(total1 + (p.together ? total2 : 0), at_once(p.shared.kernel), least(p.shared.kernel)), 128);
  } else if (any1) {
    // one CTA an SM: the number of ranges whose waves take the fewest steps of 128 rows; a CTA's start and end count as three
    long long best = 0;
    for (int s = 1; s <= 32; ++s) {
      const long long waves = (p.shared.units * s + sms - 1) / sms, steps = ((max_prefix + s - 1) / s + 127) / 128;
      const long long cost = waves * (steps + 3);
      if (s == 1 || cost < best) {
        best = cost;
        p.shared.splits = s;
      }
    }
  }
  p.shared.units *= p.shared.splits;
  p.own.units *= p.own.splits;
  p.parts = p.shared.splits + p.own.splits;
  return p;
}
