// How attention over shared prefixes is cut into CTAs (host code, no CUDA).
#pragma once
#include <algorithm>

struct PrefixPlan {
  int tile1, tile2;         // query rows of a CTA: shared part, own part
  int tiles1, splits1;      // shared rows: query tiles of a group and head, ranges that its rows are cut into
  int tiles2, splits2;      // own rows: query tiles of an item and head, ranges
  int tc;                   // the shared part runs on tcgen05: two parts of a result for every range
  int parts1, parts;        // of a result: of the shared part, and all
};

// max_group items of `rep` heads share a group's rows; `most`: query rows a CTA of the plain kernels may have; `tc`: tcgen05 may be
// used.
inline PrefixPlan prefix_plan(long long n_groups, long long max_group, long long max_prefix, long long n_items, long long max_own, int n_kv,
                              int rep, int most, bool tc, int sms) {
  PrefixPlan p{};
  const long long rows = max_group * rep;
  const auto tile = [&](long long n) { return n <= 16 || most <= 16 ? 16 : n <= 32 ? 32 : 64; };
  p.tc = tc && n_groups > 0 && rows > 64;
  p.tile1 = p.tc ? 256 : tile(rows);
  p.tile2 = tile(rep);
  p.tiles1 = n_groups > 0 ? (int)((rows + p.tile1 - 1) / p.tile1) : 0;
  p.tiles2 = max_own > 0 ? (rep + p.tile2 - 1) / p.tile2 : 0;
  const long long units1 = n_groups * n_kv * p.tiles1, units2 = max_own > 0 ? n_items * n_kv * p.tiles2 : 0;
  // cached rows that a CTA is given: what four CTAs an SM leave for each, 256 at least
  long long chunk = ((p.tc ? 0 : units1 * max_prefix) + units2 * max_own) / (4LL * sms) + 1;
  if (chunk < 256) chunk = 256;
  const auto cut = [&](long long n) { return (int)std::min(32LL, std::max(1LL, (n + chunk - 1) / chunk)); };
  p.splits1 = n_groups > 0 ? cut(max_prefix) : 0;
  p.splits2 = max_own > 0 ? cut(max_own) : 0;
  if (p.tc) {
    // one CTA an SM: the number of ranges whose waves take the fewest steps of 128 rows; a CTA's start and end count as three
    long long best = 0;
    for (int s = 1; s <= 16; ++s) {
      const long long waves = (units1 * s + sms - 1) / sms, steps = ((max_prefix + s - 1) / s + 127) / 128;
      const long long cost = waves * (steps + 3);
      if (s == 1 || cost < best) {
        best = cost;
        p.splits1 = s;
      }
    }
  }
  p.parts1 = p.tc ? 2 * p.splits1 : p.splits1;
  p.parts = p.parts1 + p.splits2;
  return p;
}
