// How attention over shared prefixes is cut into units of work (host code, no CUDA).
#pragma once
#include <algorithm>

// What goes through the shared rows, by the query rows that a group's items have at a key head: a warp for up to 24, a CTA with
// tcgen05 products for more.  Own rows are a warp's.  32-bit formats: a CTA for 16 query rows of either part.
enum : int { AP_SHARED_ROWS = 0, AP_SHARED_TC = 1, AP_SHARED_PLAIN = 2 };
constexpr int AP_WARPS_PER_SM = 8;      // that go through cached rows

struct PrefixPlan {
  int shared;               // AP_SHARED_*
  int tile1, tile2;         // query rows of a unit: shared part, own part
  int rows;                 // the most that a warp's unit has
  int tiles1, splits1;      // shared rows: query tiles of a group and head, ranges that its rows are cut into
  int tiles2, splits2;      // own rows: query tiles of an item and head, ranges
  int parts1, parts;        // of a result: of the shared part, and all
};

// max_group items of `rep` heads share a group's rows; `most`: query rows a warp may have; `wide`: 32-bit formats; `tc`: tcgen05 may be
// used.
inline PrefixPlan prefix_plan(long long n_groups, long long max_group, long long max_prefix, long long n_items, long long max_own, int n_kv,
                              int rep, int most, bool wide, bool tc, int sms) {
  PrefixPlan p{};
  const long long rows = max_group * rep;
  p.shared = wide ? AP_SHARED_PLAIN : rows <= 24 || !tc ? AP_SHARED_ROWS : AP_SHARED_TC;
  p.tile1 = p.shared == AP_SHARED_TC ? 256 : wide ? 16 : most;
  p.tile2 = wide ? 16 : most;
  p.tiles1 = n_groups > 0 ? (int)((rows + p.tile1 - 1) / p.tile1) : 0;
  p.tiles2 = max_own > 0 ? (rep + p.tile2 - 1) / p.tile2 : 0;
  const long long units1 = n_groups * n_kv * p.tiles1, units2 = max_own > 0 ? n_items * n_kv * p.tiles2 : 0;
  const auto cut = [](long long n, long long chunk, long long most) { return (int)std::min(most, std::max(1LL, (n + chunk - 1) / chunk)); };
  const bool together = p.shared != AP_SHARED_TC;
  // cached rows of a warp's unit: all of them divided by the warps; four units a warp where they are long
  const long long each = ((together ? units1 * max_prefix : 0) + units2 * max_own) / ((long long)AP_WARPS_PER_SM * sms);
  const long long chunk = each < 256 ? std::max(64LL, each) : std::max(256LL, each / 4);
  p.splits2 = max_own > 0 ? cut(max_own, chunk, 32) : 0;
  if (n_groups > 0) {
    if (together) {
      p.splits1 = cut(max_prefix, chunk, 128);
    } else {
      // one CTA an SM: the number of ranges whose waves take the fewest steps of 128 rows; a CTA's start and end count as three
      long long best = 0;
      for (int s = 1; s <= 32; ++s) {
        const long long waves = (units1 * s + sms - 1) / sms, steps = ((max_prefix + s - 1) / s + 127) / 128;
        const long long cost = waves * (steps + 3);
        if (s == 1 || cost < best) {
          best = cost;
          p.splits1 = s;
        }
      }
    }
  }
  const long long own = max_own > 0 ? std::min<long long>(rep, p.tile2) : 0;
  p.rows = (int)std::max(own, p.shared == AP_SHARED_ROWS && n_groups > 0 ? std::min<long long>(rows, p.tile1) : 0LL);
  p.parts1 = p.shared == AP_SHARED_TC ? 2 * p.splits1 : p.splits1;      // two chains a CTA
  p.parts = p.parts1 + p.splits2;
  return p;
}
