// Attention over shared cached rows in 16-bit formats for up to 16 query rows at a time: the rows of an item's own, and shared
// rows that few queries see.
//
// A unit of work is a range of one sequence's cached rows and up to 16 query rows.  A warp takes units by itself: keys and values
// are copied asynchronously into a ring of its own (16-byte pieces, exclusive-or swizzled by the row), and the ring runs on
// into the next unit (its queries with its first tile) while this one is finished, so that a unit's start costs no wait and
// short ranges stream as long ones do.  There is no barrier between warps: every unit writes a part of the result.  S = Q K^T and
// O += P V are m16n8k16 products with fp32 sums; queries, sums and weights stay in registers.  What bounds it is reading the cache.
// Descriptions of units are worked out for 32 units of a warp at once, one a lane.
//
// Rounding as in attn_prefix_mma.cu: weights are two 16-bit pieces, half queries over a bfloat16 cache too.
#include "attn_prefix_frag.cuh"
#include "flash_common.cuh"
#include "gemm.cuh"
#include "launch.cuh"

namespace {

constexpr float AR_RESCALE = 8.f;      // log2 units
constexpr int AR_WARPS = 4;

template <int D>
struct ArCfg {
  static constexpr int KEYS = D == 64 ? 32 : 16;           // of a tile
  static constexpr int STAGES = 3;
  static constexpr int PLANE = KEYS * D * 2;
  static constexpr int STAGE = 2 * PLANE;
  static constexpr int Q_BYTES = 16 * D * 2;
  static constexpr int WARP = STAGES * STAGE + Q_BYTES;
  static constexpr int SMEM = AR_WARPS * WARP;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
};

template <int D, bool HALF, bool QS>
__global__ void __launch_bounds__(AR_WARPS * 32, 2)
attn_prefix_rows_kernel(AttnPrefixArgs a, long long n_units) {
  using C = ArCfg<D>;
  constexpr int NT = C::KEYS / 8, DK = D / 16, CH = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(128) uint8_t ar_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(ar_smem)) + warp * C::WARP, q_slot = ring + C::STAGES * C::STAGE;
  const long long n_warps = (long long)gridDim.x * AR_WARPS, mine = (long long)warp * gridDim.x + blockIdx.x;
  if (mine >= n_units) return;
  const int n = (int)((n_units - mine + n_warps - 1) / n_warps);          // units of this warp

  ApWork batch;
  int batch_of = -1;
  auto unit = [&](int i) {
    if (i >> 5 != batch_of) {
      batch_of = i >> 5;
      const long long u = mine + (long long)((batch_of << 5) + lane) * n_warps;
      if (u < n_units) batch = ap_work(a, a.first_block + u, true);
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
  };
  const int col = lane % CH, row = lane / CH;      // a lane copies piece `col` of rows row, row + 32 / CH, ...
  // tile t of unit w into slot `put`, with the queries when it is the first
  auto issue = [&](const ApWork& w, int t, int put) {
    const uint32_t st = ring + put * C::STAGE;
    const size_t row0 = (((size_t)w.seq * a.n_kv + w.kvh) * (size_t)a.t_max + w.begin) * CH + col;
    const int left = w.end - w.begin - t * C::KEYS;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      const char* src = reinterpret_cast<const char*>(plane ? a.v : a.k) + row0 * 16;
#pragma unroll
      for (int i = 0; i < C::KEYS * CH / 32; ++i) {
        const int r = row + i * (32 / CH);
        const bool ok = r < left;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(st + plane * C::PLANE + r * (CH * 16) + ((col ^ (r & 7)) << 4)),
                     "l"(src + (size_t)(ok ? t * C::KEYS + r : 0) * (CH * 16)), "r"(ok ? 16 : 0) : "memory");
      }
    }
    if (t == 0) {
      const char* q = reinterpret_cast<const char*>(a.q) + col * 16;
#pragma unroll
      for (int i = 0; i < 16 * CH / 32; ++i) {
        const int r = row + i * (32 / CH), R = w.r0 + r;
        const bool ok = r < w.rows;
        const size_t at = ok ? ((size_t)(w.item0 + R / a.rep) * a.q_pitch + (size_t)(w.kvh * a.rep + R % a.rep) * D) * 2 : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_slot + r * (CH * 16) + ((col ^ (r & 7)) << 4)), "l"(q + at), "r"(ok ? 16 : 0) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto tiles_of = [&](const ApWork& w) { return (w.end - w.begin + C::KEYS - 1) / C::KEYS; };

  const float sc = fabsf(a.scale) * AP_LOG2E;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;        // a negative scale turns the queries, so that maxima are maxima
  const bool whole = a.plan.parts == 1;

  ApWork cur = unit(0), ahead = cur;       // the unit at work, and the one that tiles are asked for of
  int ahead_i = 0, ahead_t = 0;            // its number, and its next tile
  int flight = 0, put = 0, get = 0;        // tiles asked for and not used up
  for (int i = 0; i < n; ++i) {
    const int tiles = tiles_of(cur);
    // asks for tiles while there is room, up to the end of the next unit; into that (cross) only when this one's queries have
    // left their slot
    auto ask = [&](bool cross) {
      while (flight < C::STAGES) {
        if (ahead_t == tiles_of(ahead)) {
          if (!cross || ahead_i != i || i + 1 == n) break;
          ahead = unit(++ahead_i);
          ahead_t = 0;
          if (tiles_of(ahead) == 0) break;
        }
        issue(ahead, ahead_t++, put);
        put = put + 1 == C::STAGES ? 0 : put + 1;
        ++flight;
      }
    };
    uint32_t q[DK][4], ql[QS ? DK : 1][4];
    float acc[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < D / 8; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
    for (int t = 0; t < tiles; ++t) {
      __syncwarp();                        // everybody is done with the tile before, whose slot is asked for now
      ask(t > 0);
      if (flight == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else if (flight == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 2;" ::: "memory");
      static_assert(C::STAGES == 3, "waits for one to three tiles under way");
      __syncwarp();
      if (t == 0) {
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) {
          const int r = lane & 15;
          uint32_t in[4];
          am_ld4(q_slot + r * (CH * 16) + (((2 * ks + (lane >> 4)) ^ (r & 7)) << 4), in);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (QS) {
              const float2 f = unpack2_act(in[e] ^ flip, 1);
              am_split<false>(f.x, f.y, q[ks][e], ql[ks][e]);
            } else {
              q[ks][e] = in[e] ^ flip;
            }
          }
        }
        __syncwarp();
        ask(true);
      }
      const uint32_t kst = ring + get * C::STAGE, vst = kst + C::PLANE;
      get = get + 1 == C::STAGES ? 0 : get + 1;
      --flight;
      const int left = cur.end - cur.begin - t * C::KEYS;        // keys of the tile
      float s[NT][4];
#pragma unroll
      for (int e = 0; e < NT; ++e) s[e][0] = s[e][1] = s[e][2] = s[e][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DK; ++ks)
#pragma unroll
        for (int e = 0; e < NT; e += 2) {
          const int r = e * 8 + (lane & 7) + ((lane >> 4) << 3);
          uint32_t b[4];
          am_ld4(kst + r * (CH * 16) + (((2 * ks + ((lane >> 3) & 1)) ^ (r & 7)) << 4), b);
          am_mma<HALF>(s[e], q[ks], b[0], b[1]);
          am_mma<HALF>(s[e + 1], q[ks], b[2], b[3]);
          if constexpr (QS) {
            am_mma<HALF>(s[e], ql[ks], b[0], b[1]);
            am_mma<HALF>(s[e + 1], ql[ks], b[2], b[3]);
          }
        }
      const bool some = left < C::KEYS;
      if (some)
#pragma unroll
        for (int e = 0; e < NT; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (e * 8 + (lane & 3) * 2 + (j & 1) >= left) s[e][j] = -INFINITY;
      float alpha[2] = {1.f, 1.f};
      bool raise = false;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float mx = fmaxf(s[0][2 * x], s[0][2 * x + 1]);
#pragma unroll
        for (int e = 1; e < NT; ++e) mx = max3_f32(mx, s[e][2 * x], s[e][2 * x + 1]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = mx == -INFINITY ? -INFINITY : mx * sc;
        if (mx > m[x] + AR_RESCALE || (m[x] == -INFINITY && mx > -INFINITY)) {
          alpha[x] = m[x] == -INFINITY ? 0.f : ex2_fast(m[x] - mx);
          raise = true;
          m[x] = mx;
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
        l[0] *= alpha[0];
        l[1] *= alpha[1];
#pragma unroll
        for (int e = 0; e < D / 8; ++e) {
          acc[e][0] *= alpha[0]; acc[e][1] *= alpha[0];
          acc[e][2] *= alpha[1]; acc[e][3] *= alpha[1];
        }
      }
      const float safe[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int e = 0; e < NT; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float p = ex2_fast(fmaf(s[e][j], sc, -safe[j >> 1]));
          if (some && e * 8 + (lane & 3) * 2 + (j & 1) >= left) p = 0.f;     // also where the scale is 0
          l[j >> 1] += p;
          s[e][j] = p;
        }
#pragma unroll
      for (int kk = 0; kk < C::KEYS / 16; ++kk) {
        uint32_t hi[4], lo[4];
        am_split<HALF>(s[2 * kk][0], s[2 * kk][1], hi[0], lo[0]);
        am_split<HALF>(s[2 * kk][2], s[2 * kk][3], hi[1], lo[1]);
        am_split<HALF>(s[2 * kk + 1][0], s[2 * kk + 1][1], hi[2], lo[2]);
        am_split<HALF>(s[2 * kk + 1][2], s[2 * kk + 1][3], hi[3], lo[3]);
        const int r = kk * 16 + (lane & 15);
#pragma unroll
        for (int dt = 0; dt < DK; ++dt) {
          uint32_t b[4];
          am_ld4t(vst + r * (CH * 16) + (((2 * dt + (lane >> 4)) ^ (r & 7)) << 4), b);
          am_mma<HALF>(acc[2 * dt], hi, b[0], b[1]);
          am_mma<HALF>(acc[2 * dt + 1], hi, b[2], b[3]);
          am_mma<HALF>(acc[2 * dt], lo, b[0], b[1]);
          am_mma<HALF>(acc[2 * dt + 1], lo, b[2], b[3]);
        }
      }
    }
    // the unit's part of the result
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      const int r = (lane >> 2) + 8 * x, R = cur.r0 + r;
      if (r >= cur.rows) continue;
      const int item = cur.item0 + R / a.rep;
      const long long ih = (long long)item * a.n_heads + cur.kvh * a.rep + R % a.rep;
      if (whole) {
        const bool none = l[x] == 0.f || (a.item_skip && a.item_skip[item]);
        const float inv = 1.f / l[x];
#pragma unroll
        for (int e = 0; e < D / 8; ++e)
          ap_store2(a.out, (size_t)ih * D + e * 8 + (lane & 3) * 2, none ? 0.f : acc[e][2 * x] * inv, none ? 0.f : acc[e][2 * x + 1] * inv, a.act_fmt);
      } else {
        float* to = ap_record(a, ih, cur.part);
        if (tiles > 0)
#pragma unroll
          for (int e = 0; e < D / 8; ++e) *reinterpret_cast<float2*>(to + e * 8 + (lane & 3) * 2) = make_float2(acc[e][2 * x], acc[e][2 * x + 1]);
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m[x], l[x]);
      }
    }
    if (i + 1 < n) {
      if (ahead_i == i) {
        ahead = unit(++ahead_i);
        ahead_t = 0;
      }
      cur = ahead;
    }
  }
}

template <int D, bool HALF, bool QS>
cudaError_t ar_launch(const AttnPrefixArgs& a, long long units, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = arcb_opt_in_smem(attn_prefix_rows_kernel<D, HALF, QS>, ArCfg<D>::SMEM, done);
  if (e != cudaSuccess) return e;
  const long long most = 2LL * arcb_num_sms();
  return arcb_launch(attn_prefix_rows_kernel<D, HALF, QS>, dim3((unsigned)(units < most ? units : most)), dim3(AR_WARPS * 32), ArCfg<D>::SMEM, stream, a, units);
}

}  // namespace

cudaError_t arcb_attn_prefix_rows(const AttnPrefixArgs& a, long long units, cudaStream_t stream) {
  if (a.kv_fmt == 1) return a.dim == 64 ? ar_launch<64, true, false>(a, units, stream) : ar_launch<128, true, false>(a, units, stream);
  if (a.act_fmt == 1) return a.dim == 64 ? ar_launch<64, false, true>(a, units, stream) : ar_launch<128, false, true>(a, units, stream);
  return a.dim == 64 ? ar_launch<64, false, false>(a, units, stream) : ar_launch<128, false, false>(a, units, stream);
}
