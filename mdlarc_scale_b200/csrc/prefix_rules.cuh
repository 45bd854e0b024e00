// How attention over shared prefixes is cut into CTAs (host code, no CUDA).
#pragma once
#include <algorithm>

struct PrefixPlan {
  int tile1, tile2;         // query rows of a CTA
  int tiles1, splits1;      // shared rows: query tiles of a group and head, ranges that its rows are cut into
  int tiles2, splits2;      // own rows: query tiles of an item and head, ranges
  int parts;                // of a result: splits1 + splits2
};

// max_group items of `rep` heads share a group's rows; `most`: query rows a CTA may have.
inline PrefixPlan prefix_plan(long long n_groups, long long max_group, long long max_prefix, long long n_items, long long max_own, int n_kv,
                              int rep, int most, int sms) {
  PrefixPlan p{};
  const auto tile = [&](long long n) { return n <= 16 || most <= 16 ? 16 : n <= 32 ? 32 : 64; };
  p.tile1 = tile(max_group * rep);
  p.tile2 = tile(rep);
  const long long rows = max_group * rep;
  p.tiles1 = n_groups > 0 ? (int)((rows + p.tile1 - 1) / p.tile1) : 0;
  p.tiles2 = max_own > 0 ? (rep + p.tile2 - 1) / p.tile2 : 0;
  const long long units1 = n_groups * n_kv * p.tiles1, units2 = max_own > 0 ? n_items * n_kv * p.tiles2 : 0;
  // cached rows that a CTA is given: what four CTAs an SM leave for each, 256 at least
  long long chunk = (units1 * max_prefix + units2 * max_own) / (4LL * sms) + 1;
  if (chunk < 256) chunk = 256;
  const auto cut = [&](long long n) { return (int)std::min(32LL, std::max(1LL, (n + chunk - 1) / chunk)); };
  p.splits1 = n_groups > 0 ? cut(max_prefix) : 0;
  p.splits2 = max_own > 0 ? cut(max_own) : 0;
  p.parts = p.splits1 + p.splits2;
  return p;
}
