// Attention over shared cached rows in 16-bit formats for up to eight query rows at a time: the rows of an item's own, and shared
// rows that few queries see.
//
// A unit of work is a range of one sequence's cached rows and up to eight query rows.  A warp takes units by itself: keys and values
// come by cp.async into a ring of its own (rows of 128 bytes, 16-byte pieces exclusive-or swizzled), and the ring runs on into the
// next unit (its queries with its first tile) while this one is finished, so that a unit's start costs no wait and short ranges
// stream as long ones do.  There is no barrier between warps: every unit writes a part of the result, which a second kernel joins.
// Where the rows of a whole group are few, the eight warps of one CTA take all units of a (group, key head) and join them in
// shared memory: one launch in place of two and no parts in memory.
// Descriptions of units are worked out for 32 units of a warp at once, one a lane.
//
// The products are transposed, so that the eight columns of m16n8k16 are queries: S^T = K Q^T (16 keys a product) and O^T += V^T P^T
// (16 value columns a product); weights change from the first one's result to the second one's operand by 8 x 8 transpositions
// in the warp.  These products are slow here, 14 cycles each, and with 16 queries a product most of them would be padding.  What
// bounds it is reading the cache: 64 x 20 groups of eight queries over 1193 shared rows and 300 of each one's own, heads of 64 (647 MB):
// 121 us, 5.3 TB/s, the join of the parts 6 more.
//
// Rounding: a weight enters the product as two 16-bit pieces (p = hi + lo), since one piece alone would be as far off as the
// output's own rounding; half queries over a bfloat16 cache are two bfloat16 pieces, which is exact.  With up to four query rows the
// weights' pieces are columns of their own and cost nothing.  Maxima, sums and all partial results are fp32.  A range's reference
// is raised only when its maximum grows by 2^8; in half it is 2^7 below the maximum, so that weights are up to 2^15 and end at 2^-24
// of it: weights down to 2^-32 of a range's largest one count.
#include "attn_prefix_frag.cuh"
#include "flash_common.cuh"
#include "gemm.cuh"
#include "launch.cuh"

using namespace sm100;

namespace {

constexpr float AR_RESCALE = 8.f, AR_BELOW = 7.f;      // log2 units
constexpr int AR_WARPS = 4;      // of a CTA; AP_GROUP_WARPS of one that takes a group

template <int D>
struct ArCfg {
  static constexpr int CTAS = 3;           // of an SM
  static constexpr int KEYS = D == 64 ? 32 : 16;           // of a tile
  static constexpr int STAGES = 2;
  static constexpr int BOX = KEYS * 128;
  static constexpr int PLANE = KEYS * D * 2;
  static constexpr int STAGE = 2 * PLANE;
  static constexpr int Q_BYTES = 8 * D * 2;
  static constexpr int WARP = STAGES * STAGE + Q_BYTES;
  static_assert(WARP % 128 == 0 && BOX % 128 == 0, "an exclusive-or of an address is one of its piece of 128 bytes");
  static constexpr int SMEM = AR_WARPS * WARP;
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs of an SM");
};

// What a warp keeps from unit to unit.  GROUP: the units are those of group g and key head kvh, the shared ranges and then the items'.
template <int D, bool GROUP>
struct ArWarp {
  using C = ArCfg<D>;
  static constexpr int CH = D / 8;         // 16-byte pieces of a row
  const AttnPrefixArgs& a;
  long long first, stride, n_units;        // this warp's units
  int n, lane;
  uint32_t ring, q_slot, to;               // `to`: where a lane's first piece of a tile goes
  ApWork batch;
  int batch_of;
  ApWork ahead;                            // the unit that tiles are asked for of, its number, its tiles that have not been,
  int ahead_i, ahead_left, rows_left;      // the rows from the next one on, and where they are
  const char* from[2];
  int flight, put, get;                    // tiles asked for and not used up
  int g, kvh, item0, items;                // GROUP: and its items, max_group of them at a time
  float* records;                          // GROUP: [query row][part][D + AP_PAD]

  __device__ __forceinline__ ApWork work(long long u) const {
    if constexpr (GROUP) {
      const int splits = a.plan.shared.splits, own = (int)u - splits;
      if (own < 0) {
        ApWork w = ap_work(a, ((long long)g * a.n_kv + kvh) * splits + u, true);
        w.item0 = item0;
        w.rows = items * a.rep;
        return w;
      }
      const int item = own / a.plan.own.splits;
      if (item >= items) return ApWork{};
      return ap_work(a, a.plan.shared.units + ((long long)(item0 + item) * a.n_kv + kvh) * a.plan.own.splits + own % a.plan.own.splits, true);
    } else {
      return ap_work(a, a.first_block + u, true);
    }
  }

  __device__ __forceinline__ ApWork unit(int i) {
    if (i >> 5 != batch_of) {
      batch_of = i >> 5;
      const long long u = first + (long long)((batch_of << 5) + lane) * stride;
      if (u < n_units) batch = work(u);
    }
    ApWork w;
    const int from = i & 31;
    w.item0 = __shfl_sync(0xffffffffu, batch.item0, from);
    w.r0 = __shfl_sync(0xffffffffu, batch.r0, from);
    w.rows = __shfl_sync(0xffffffffu, batch.rows, from);
    w.kvh = __shfl_sync(0xffffffffu, batch.kvh, from);
    w.seq = __shfl_sync(0xffffffffu, batch.seq, from);
    w.begin = __shfl_sync(0xffffffffu, batch.begin, from);
    w.end = __shfl_sync(0xffffffffu, batch.end, from);
    w.part = __shfl_sync(0xffffffffu, batch.part, from);
    if (w.rows <= 0) w.end = w.begin;
    return w;
  }
  static __device__ __forceinline__ int tiles_of(const ApWork& w) { return (w.end - w.begin + C::KEYS - 1) / C::KEYS; }
  // query row r of a unit
  __device__ __forceinline__ const char* query(const ApWork& w, int r) const {
    const int R = w.r0 + r;
    return reinterpret_cast<const char*>(a.q) + ((size_t)(w.item0 + R / a.rep) * a.q_pitch + (size_t)(w.kvh * a.rep + R % a.rep) * D) * 2;
  }
  __device__ __forceinline__ void look_at(const ApWork& w) {
    ahead = w;
    ahead_left = tiles_of(w);
    rows_left = w.end - w.begin;
    const size_t at = (((size_t)w.seq * a.n_kv + w.kvh) * (size_t)a.t_max + w.begin + lane / CH) * (D * 2) + (lane % CH) * 16;
    from[0] = reinterpret_cast<const char*>(a.k) + at;
    from[1] = reinterpret_cast<const char*>(a.v) + at;
  }
  // the next tile into slot `put`, with the unit's queries when it is the first; rows behind the end become zeros
  __device__ __forceinline__ void issue() {
    constexpr int STEP = 32 / CH;          // rows of a pass; a lane has one 16-byte piece of each
    const uint32_t st = ring + put * C::STAGE + to;
    if (rows_left >= C::KEYS) {
#pragma unroll
      for (int plane = 0; plane < 2; ++plane)
#pragma unroll
        for (int i = 0; i < C::KEYS / STEP; ++i)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((st ^ piece(i)) + plane * C::PLANE + i * STEP * 128), "l"(from[plane] + i * STEP * (D * 2)) : "memory");
    } else {
#pragma unroll
      for (int plane = 0; plane < 2; ++plane)
#pragma unroll
        for (int i = 0; i < C::KEYS / STEP; ++i) {
          const bool ok = lane / CH + i * STEP < rows_left;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((st ^ piece(i)) + plane * C::PLANE + i * STEP * 128),
                       "l"(ok ? from[plane] + i * STEP * (D * 2) : reinterpret_cast<const char*>(a.k)), "r"(ok ? 16 : 0) : "memory");
        }
    }
    if (ahead_left == tiles_of(ahead)) {
      for (int r = lane / CH; r < ahead.rows; r += STEP)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(q_slot + r * (D * 2) + (lane % CH) * 16), "l"(query(ahead, r) + (lane % CH) * 16) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    from[0] += C::KEYS * D * 2;
    from[1] += C::KEYS * D * 2;
    rows_left -= C::KEYS;
    --ahead_left;
    put = put + 1 == C::STAGES ? 0 : put + 1;
    ++flight;
  }
  // the swizzle of row lane / CH + i STEP beside that of row lane / CH
  static __device__ __forceinline__ uint32_t piece(int i) { return ((i * (32 / CH)) & 7) << 4; }
  // Asks for tiles while there is room, up to the end of the unit behind unit i; into that (cross) only when the queries of
  // unit i have left their slot.
  __device__ __forceinline__ void ask(int i, bool cross) {
    while (flight < C::STAGES) {
      if (ahead_left == 0) {
        if (!cross || ahead_i != i || i + 1 == n) break;
        look_at(unit(++ahead_i));
        if (ahead_left == 0) break;
      }
      issue();
    }
  }
};

// One unit.  PAIR: up to four query rows; columns 4 to 7 of the products are second pieces of weights.
template <int D, bool HALF, bool QS, bool PAIR, bool GROUP>
__device__ __forceinline__ void ar_unit(ArWarp<D, GROUP>& s, const ApWork& w, int i) {
  using C = ArCfg<D>;
  constexpr int DK = D / 16, MT = C::KEYS / 16;
  constexpr float BELOW = HALF ? AR_BELOW : 0.f;
  const AttnPrefixArgs& a = s.a;
  const int lane = s.lane;
  // A negative scale turns the queries, so that maxima are maxima; one of 0 makes them 0, since 0 times -inf is no score.
  const float sc = a.scale == 0.f ? 1.f : fabsf(a.scale) * AP_LOG2E;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, kept = a.scale == 0.f ? 0u : 0xffffffffu;
  const int tiles = s.tiles_of(w);
  // A lane has queries (lane % 4) * 2 and the next one (PAIR: of the first four), and keys or value columns lane / 4 and that plus 8 of
  // every 16.
  uint32_t q[DK][2], q2[QS ? DK : 1][2];
  float acc[DK][4], m[2] = {-INFINITY, -INFINITY}, off[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};     // off: what is taken off a score, -m or 0
#pragma unroll
  for (int e = 0; e < DK; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
  auto keep_query = [&](int ks, int y, uint32_t raw) {
    raw = (raw ^ flip) & kept;
    if constexpr (QS) {
      const float2 f = unpack2_act(raw, 1);
      am_split<false>(f.x, f.y, q[ks][y], q2[ks][y]);
    } else {
      q[ks][y] = raw;
    }
  };
  // Pieces of matrix loads: row (lane % 16) and row (lane % 8) + 8 (lane / 16) of 16; 16-byte piece 2 ks + h lies at (2 ks + h) ^ row % 8,
  // which is one exclusive-or of the address with 32 ks.
  const uint32_t k_at = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_at = ((lane & 7) + ((lane >> 4) << 3)) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  for (int t = 0; t < tiles; ++t) {
    __syncwarp();                          // everybody is done with the tile before, whose slot is asked for now
    s.ask(i, t > 0);
    if (s.flight == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (s.flight == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
    static_assert(C::STAGES <= 3, "waits for one to three tiles under way");
    __syncwarp();
    if (t == 0) {
      const int r = min(lane & (PAIR ? 3 : 7), w.rows - 1);      // rows that do not exist are as the last one
#pragma unroll
      for (int ks = 0; ks < DK; ks += 2) {
        uint32_t in[4];
        am_ld4(s.q_slot + r * (D * 2) + ((2 * ks + (lane >> 3)) << 4), in);
        keep_query(ks, 0, in[0]);
        keep_query(ks, 1, in[1]);
        keep_query(ks + 1, 0, in[2]);
        keep_query(ks + 1, 1, in[3]);
      }
      __syncwarp();
      s.ask(i, true);
    }
    const uint32_t slot = s.ring + s.get * C::STAGE, kst = slot + k_at, vst = slot + C::PLANE + v_at;
    s.get = s.get + 1 == C::STAGES ? 0 : s.get + 1;
    --s.flight;
    const int left = w.end - w.begin - t * C::KEYS;        // keys of the tile
    const bool some = left < C::KEYS;
    float p[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) p[mt][0] = p[mt][1] = p[mt][2] = p[mt][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) {
      const uint32_t at = (kst ^ ((ks & 3) << 5)) + (ks >> 2) * C::BOX;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t k[4];
        am_ld4(at + mt * (16 * 128), k);
        am_mma<HALF>(p[mt], k, q[ks][0], q[ks][1]);
        if constexpr (QS) am_mma<HALF>(p[mt], k, q2[ks][0], q2[ks][1]);
      }
    }
    if (some) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (mt * 16 + (lane >> 2) + (j >> 1) * 8 >= left) p[mt][j] = -INFINITY;
    }
    // the lanes' own maxima tell whether any reference has to be raised; only then are they exchanged
    float top[2];
    bool raise = t == 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float mx = fmaxf(p[0][x], p[0][2 + x]);
#pragma unroll
      for (int mt = 1; mt < MT; ++mt) mx = max3_f32(mx, p[mt][x], p[mt][2 + x]);
      top[x] = mx;
      raise |= mx * sc > m[x] + (AR_RESCALE + BELOW);
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float mx = top[x];
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx = fmaxf(fmaf(mx, sc, -BELOW), m[x]);
        if (mx == -INFINITY) continue;
        const float alpha = m[x] == -INFINITY ? 0.f : ex2_fast(m[x] - mx);
        m[x] = mx;
        off[x] = -mx;
        l[x] *= alpha;
#pragma unroll
        for (int e = 0; e < DK; ++e) {
          acc[e][x] *= alpha;
          acc[e][2 + x] *= alpha;
        }
      }
    }
    uint32_t hi[MT][2], lo[PAIR ? 1 : MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float e0 = ex2_fast(fmaf(p[mt][2 * y], sc, off[0])), e1 = ex2_fast(fmaf(p[mt][2 * y + 1], sc, off[1]));
        l[0] += e0;
        l[1] += e1;
        uint32_t h, o;
        am_split<HALF>(e0, e1, h, o);
        hi[mt][y] = am_transpose(PAIR && (lane & 2) ? o : h);
        if constexpr (!PAIR) lo[mt][y] = am_transpose(o);
      }
#pragma unroll
    for (int dt = 0; dt < DK; ++dt) {
      const uint32_t at = (vst ^ ((dt & 3) << 5)) + (dt >> 2) * C::BOX;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t v[4];
        am_ld4t(at + mt * (16 * 128), v);
        am_mma<HALF>(acc[dt], v, hi[mt][0], hi[mt][1]);
        if constexpr (!PAIR) am_mma<HALF>(acc[dt], v, lo[mt][0], lo[mt][1]);
      }
    }
  }
  // The unit's part of the result: eight lanes have eight neighbouring value columns of a query.
  const bool whole = !GROUP && !a.plan.joined;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (x >= w.rows) break;
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], o);
    const int r = (lane & (PAIR ? 1 : 3)) * 2 + x;
    const bool in = r < w.rows && !(PAIR && (lane & 2));
    const int R = w.r0 + (in ? r : 0), item = w.item0 + R / a.rep;
    const long long ih = (long long)item * a.n_heads + w.kvh * a.rep + R % a.rep;
    const float inv = l[x] == 0.f || (whole && in && a.item_skip && a.item_skip[item]) ? 0.f : 1.f / l[x];
    float* to = whole ? nullptr
                : GROUP ? s.records + (((item - s.item0) * a.rep + R % a.rep) * a.plan.parts + w.part) * (D + AP_PAD) + (lane >> 2)
                        : ap_record(a, ih, w.part) + (lane >> 2);
#pragma unroll
    for (int e = 0; e < DK; ++e)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float v = acc[e][2 * y + x];
        if constexpr (PAIR) v += __shfl_xor_sync(0xffffffffu, v, 2);
        if (!in) continue;
        if (whole) ap_store1(a.out, (size_t)ih * D + e * 16 + y * 8 + (lane >> 2), inv == 0.f ? 0.f : v * inv, a.act_fmt);
        else if (tiles > 0) to[e * 16 + y * 8] = v;
      }
    if (in && !whole && lane < 4) *reinterpret_cast<float2*>(to + D) = make_float2(m[x], l[x]);
  }
}

// A query row's parts, by one warp.
template <int D>
__device__ __forceinline__ void ar_join(const AttnPrefixArgs& a, const float* rec, int item, int head, int lane) {
  if (lane * 4 >= D) return;
  const int n = a.plan.parts;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < n; ++s) m = fmaxf(m, rec[s * (D + AP_PAD) + D]);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < n; ++s) {
    const float* part = rec + s * (D + AP_PAD);
    const float2 ml = *reinterpret_cast<const float2*>(part + D);
    const float f = exp2f(ml.x - (m == -INFINITY ? 0.f : m));
    l += ml.y * f;                         // scores that are no numbers leave no maximum, but no number as their sum
    if (ml.x == -INFINITY) continue;       // an empty part's sums count for nothing, whatever they are
    const float4 v = *reinterpret_cast<const float4*>(part + lane * 4);
    sum.x += v.x * f; sum.y += v.y * f; sum.z += v.z * f; sum.w += v.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const bool none = l == 0.f || (a.item_skip && a.item_skip[item]);
  sum = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
  ap_store4(a.out, ((size_t)item * a.n_heads + head) * D + lane * 4, sum, a.act_fmt);
}

template <int D, bool HALF, bool QS, bool GROUP>
__global__ void __launch_bounds__((GROUP ? AP_GROUP_WARPS : AR_WARPS) * 32, GROUP ? 1 : ArCfg<D>::CTAS)
attn_prefix_rows_kernel(AttnPrefixArgs a, long long n_units) {
  using C = ArCfg<D>;
  constexpr int W = GROUP ? AP_GROUP_WARPS : AR_WARPS;
  pdl_launch_dependents();
  if (!a.beside) pdl_wait();
  extern __shared__ __align__(128) uint8_t ar_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long stride = GROUP ? W : (long long)gridDim.x * W, first = GROUP ? warp : (long long)warp * gridDim.x + blockIdx.x;
  if (!GROUP && first >= n_units) {
    if (a.beside) pdl_wait();
    return;
  }
  const uint32_t base = smem_u32(ar_smem), ring = base + warp * C::WARP;
  constexpr int CH = D / 8;
  const int row = lane / CH, col = lane % CH;
  ArWarp<D, GROUP> s{a, first, stride, n_units, (int)((n_units - first + stride - 1) / stride), lane, ring, ring + C::STAGES * C::STAGE,
                     (uint32_t)((col >> 3) * C::BOX + row * 128 + (((col & 7) ^ (row & 7)) << 4))};
  s.batch_of = -1;
  s.flight = s.put = s.get = s.ahead_i = 0;
  int behind = 0;
  if constexpr (GROUP) {
    s.g = (int)blockIdx.x / a.n_kv;
    s.kvh = (int)blockIdx.x % a.n_kv;
    const ApWork all = ap_work(a, (long long)blockIdx.x * a.plan.shared.splits, false);
    s.item0 = all.item0;
    s.items = max(all.rows, 0) / a.rep;
    s.records = reinterpret_cast<float*>(ar_smem + W * C::WARP);
    behind = all.behind;
  }
  for (;;) {
    if (s.n > 0) {
      ApWork w = s.unit(0);
      s.look_at(w);
      for (int i = 0; i < s.n; ++i) {
        if (w.rows <= 4) ar_unit<D, HALF, QS, true>(s, w, i);
        else ar_unit<D, HALF, QS, false>(s, w, i);
        if (i + 1 < s.n) {
          if (s.ahead_i == i) s.look_at(s.unit(++s.ahead_i));
          w = s.ahead;
        }
      }
    }
    if constexpr (!GROUP) break;
    __syncthreads();
    for (int r = warp; r < s.items * a.rep; r += W)
      ar_join<D>(a, s.records + r * a.plan.parts * (D + AP_PAD), s.item0 + r / a.rep, s.kvh * a.rep + r % a.rep, lane);
    if (behind <= 0) break;
    __syncthreads();               // a group of more items than it may have, which see their own rows alone: the next ones
    s.item0 += s.items;
    s.items = min(behind, a.max_group);
    behind -= s.items;
    s.batch_of = -1;
    s.ahead_i = 0;
  }
  if (a.beside) pdl_wait();      // this launch's end is the other's too
}

template <int D, bool HALF, bool QS, bool GROUP>
int ar_start(const AttnPrefixArgs& a, long long ctas, long long units, size_t smem, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const auto kernel = attn_prefix_rows_kernel<D, HALF, QS, GROUP>;
  const size_t most = GROUP ? AP_GROUP_WARPS * ArCfg<D>::WARP + 8 * AP_GROUP_WARPS * (D + AP_PAD) * 4 : smem;
  const cudaError_t e = arcb_opt_in_smem(kernel, (int)most, done);
  if (e != cudaSuccess) return (int)e;
  const dim3 grid((unsigned)ctas), block((GROUP ? AP_GROUP_WARPS : AR_WARPS) * 32);
  return (int)(a.beside ? ap_launch_beside(kernel, grid, block, smem, stream, a, units) : arcb_launch(kernel, grid, block, smem, stream, a, units));
}

template <int D, bool HALF, bool QS>
int ar_launch(const AttnPrefixArgs& a, long long units, cudaStream_t stream) {
  using C = ArCfg<D>;
  if (a.plan.grouped) {
    const long long tasks = a.plan.shared.splits + (long long)a.max_group * a.plan.own.splits;
    const size_t records = (size_t)a.max_group * a.rep * a.plan.parts * (D + AP_PAD) * 4;
    return ar_start<D, HALF, QS, true>(a, (long long)a.n_groups * a.n_kv, tasks, AP_GROUP_WARPS * C::WARP + records, stream);
  }
  const long long most = (long long)C::CTAS * arcb_num_sms();
  return ar_start<D, HALF, QS, false>(a, units < most ? units : most, units, C::SMEM, stream);
}
}  // namespace

int arcb_attn_prefix_rows(const AttnPrefixArgs& a, long long units, cudaStream_t stream) {
  if (a.kv_fmt == 1) return a.dim == 64 ? ar_launch<64, true, false>(a, units, stream) : ar_launch<128, true, false>(a, units, stream);
  if (a.act_fmt == 1) return a.dim == 64 ? ar_launch<64, false, true>(a, units, stream) : ar_launch<128, false, true>(a, units, stream);
  return a.dim == 64 ? ar_launch<64, false, false>(a, units, stream) : ar_launch<128, false, false>(a, units, stream);
}
