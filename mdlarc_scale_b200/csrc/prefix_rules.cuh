// How attention over shared prefixes is cut into units of work (host code, no CUDA), and what indices from the device may be.
#pragma once
#include <algorithm>

#ifdef __CUDACC__
#define AP_RULE __host__ __device__ inline
#else
#define AP_RULE inline
#endif

// How many rows [begin, end) of sequence seq are, -1 where some are outside the cache.  The ends are looked at before they are
// subtracted: they may be any 32 bits.
AP_RULE int ap_row_count(int begin, int end, int seq, int n_seqs, int t_max) {
  if (end <= begin) return 0;
  return begin < 0 || end > t_max || seq < 0 || seq >= n_seqs ? -1 : end - begin;
}

// Kernels, by the query rows of a unit: a warp for up to 8, a CTA for up to 64, a CTA with tcgen05 products for up to 256; in 32-bit
// formats a warp for up to 4, a CTA for up to 64.
enum : int { AP_ROWS = 0, AP_TILES = 1, AP_TC = 2, AP_F32_FEW = 3, AP_F32 = 4 };

constexpr int AP_GROUP_WARPS = 8;      // of a CTA that takes a group

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
  int grouped;              // a CTA has all units of a (group, key head) and joins them itself
  int parts;                // of a result
  int joined;               // a last kernel makes results of them; else there is one, or a group's CTA has joined them
};

// `rows` query rows at each of `heads` (groups or items) x n_kv; `tc`: tcgen05 may be used.
inline PrefixPart prefix_part(long long heads, long long rows, int n_kv, bool wide, bool tc) {
  PrefixPart p{};
  p.kernel = wide ? (rows <= 4 ? AP_F32_FEW : AP_F32) : rows <= 8 ? AP_ROWS : rows <= 64 || !tc ? AP_TILES : AP_TC;
  p.tile = p.kernel == AP_F32_FEW ? (rows <= 2 ? (int)std::max(1LL, rows) : 4) : p.kernel == AP_ROWS ? 8 : p.kernel == AP_TC ? 256 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  p.tiles = (int)((rows + p.tile - 1) / p.tile);
  p.units = heads * n_kv * p.tiles;
  return p;
}
// Ranges for `rows` cached rows where every slot of the GPU has `each` rows to read.  Up to 1024, what runs at once gets one range each,
// rounded so that no few are left for a second wave (64 items x 8 key heads of 500 rows in three ranges for 1776 warps: 60 us with
// all that goes with it, 66 in four).  Above, up to four a slot, so that lengths that differ even out, none under 1024 rows: five
// tokens of 24 sequences over 4096 rows in four ranges 76 us, in eight 84; 33 items of 777 rows at most in one 133, in four 153; but
// eight samples over 1193 rows, 1280 units, in two 124 and in one 125.
inline int prefix_cut(long long rows, long long each, long long least, long long most) {
  const long long fewest = (rows + least - 1) / least;
  const long long s = each <= 1024 ? rows / std::max(1LL, each) : (rows + std::max(1024LL, each / 4) - 1) / std::max(1024LL, each / 4);
  return (int)std::min(most, std::max(1LL, std::min(fewest, s)));
}

// max_group items of `rep` heads share a group's rows.
inline PrefixPlan prefix_plan(long long n_groups, long long max_group, long long max_prefix, long long n_items, long long max_own, int n_kv,
                              int rep, int dim, bool wide, bool tc, int sms) {
  PrefixPlan p{};
  p.shared = prefix_part(n_groups, n_groups > 0 ? max_group * rep : 0, n_kv, wide, tc);
  p.own = prefix_part(n_items, max_own > 0 ? rep : 0, n_kv, wide, false);
  const bool any1 = n_groups > 0, any2 = max_own > 0;
  p.together = any1 && any2 && p.shared.kernel == p.own.kernel && (!wide || p.shared.tile == p.own.tile);
  const long long total1 = p.shared.units * max_prefix, total2 = p.own.units * max_own;
  // Units of an SM at once.  Three of four CTAs that would fit, so that own rows run beside them (16 samples: 27.6 us, 31.2 at four); in
  // 32 bits what registers and shared memory hold (16 x 20 items of 1000 rows: 71 us at 8 warps, 81 at 12).
  const auto slots = [&](const PrefixPart& part) {
    const int k = part.kernel;
    return (long long)sms * (k == AP_ROWS ? 12 : k == AP_F32_FEW ? 8 : k == AP_TILES ? 3 : dim == 128 || part.tile == 64 ? 2 : 4);
  };
  const auto least = [](int kernel) { return kernel == AP_TILES ? 256LL : 64LL; };
  if (any2) p.own.splits = prefix_cut(max_own, (total2 + (p.together ? total1 : 0)) / slots(p.own), least(p.own.kernel), 32);
  if (any1 && p.shared.kernel != AP_TC) {
    p.shared.splits = prefix_cut(max_prefix, (total1 + (p.together ? total2 : 0)) / slots(p.shared), least(p.shared.kernel), 128);
  } else if (any1) {
    // One CTA an SM: the number of ranges whose waves take the fewest steps of 128 rows.  A CTA's start and end count as eight, what a
    // range's results are written and joined for as their bytes over 10^7.  Groups differ in length: half of the cost is that of
    // waves that end on the average unit.
    const double joined = 2.0 * n_items * n_kv * rep * (dim + 4) * 4 / 1e7;
    double best = 0;
    for (int s = 1; s <= 32; ++s) {
      const long long steps = ((max_prefix + s - 1) / s + 127) / 128;
      double waves = (double)((p.shared.units * s + sms - 1) / sms);
      if (n_groups > 1) waves = (waves + (double)(p.shared.units * s) / sms + 0.5) / 2;
      const double cost = waves * (steps + 8) + s * joined;
      if (s == 1 || cost < best) {
        best = cost;
        p.shared.splits = s;
      }
    }
  }
  // A CTA of eight warps for a whole group, a warp a range or an item, where no warp gets more than 64 rows and no SM a second CTA:
  // two samples of a prompt of 190 rows 5.8 us, 8.2 in two launches, four 6.2 and 8.3, and a launch and its scratch less on
  // the host (a call of two samples 13 us in place of 19).  With a second unit for some of the warps it was slower (eight samples: 10.8 us, 7.9).
  const long long ranges = AP_GROUP_WARPS - max_group;
  if (p.together && p.shared.kernel == AP_ROWS && p.shared.tiles == 1 && n_groups * n_kv <= sms && max_prefix <= 64 * ranges && max_own <= 64) {
    p.grouped = 1;
    p.own.splits = 1;
    p.shared.splits = (int)std::min(ranges, (max_prefix + 31) / 32);
  }
  p.shared.units *= p.shared.splits;
  p.own.units *= p.own.splits;
  p.parts = p.shared.splits + p.own.splits;
  p.joined = !p.grouped && (p.parts > 1 || p.shared.kernel == AP_TC);      // the tcgen05 kernel writes parts alone
  return p;
}
