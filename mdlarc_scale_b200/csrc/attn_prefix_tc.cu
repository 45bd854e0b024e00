// Attention over shared cached rows for many query rows of a group: tcgen05 products with their sums in tensor memory.
//
// A CTA has up to 256 query rows of one (group, key head) as two tiles of 128, A and B, and goes through a range of cached rows
// 128 at a time.  With up to 128 rows B has the same queries as A and takes every other key tile, so that there are always two
// chains (scores, softmax, weights, values) of which one is in the tensor core while the other is at its exponentials.
//   warp 0        TMA: key and value tiles as 128 x 64 boxes with the 128-byte swizzle, rings shared by A and B; value rows
//                 behind the end of the last tile are set to zero: a weight of 0 does not hide a NaN
//   warp 1        products of A and of B in turn: O += P V with P read from TMEM, then the next S = Q K^T (128 TMEM columns)
//   warps 4-11    a thread a query row: maxima, exponentials, row sums, P over the row's own score columns.  (Two threads a row
//                 had to exchange maxima in every tile and took twice the instructions.)
// Maxima, sums and results are fp32.  A row's reference is raised only when the sum of a tile's weights against its maximum passes
// 2^12; in half it is 2^3 below the maximum, so that weights are up to 2^15 and end at 2^-24 of it: weights down to 2^-28 of a
// range's largest one count.  Half queries over a bfloat16 cache are two bfloat16 pieces (exact).  Weights are two 16-bit pieces in every format (half a
// step of the type squared of a weight off): one is half a step off, which adds up to half a step of sum p |v|, more than the output's
// own rounding without limit where values cancel, and 1.4 times its error on random ones (200 us in place of the 256 below).
//
// What bounds it: the chain of a tile (scores, exponentials, weights to TMEM, values, the next scores), of which two overlap.  1024
// query rows x 32768 cached rows x 8 key heads of 128 in half (138 GFLOP, 206 with the second pieces): 256 us with own rows and join.
#include <type_traits>

#include "attn_prefix_impl.cuh"
#include "flash_common.cuh"
#include "gemm.cuh"
#include "launch.cuh"

using namespace sm100;

namespace {

constexpr int AT_ROWS = 128, AT_KEYS = 128, AT_THREADS = 384;
constexpr float AT_RAISE = 4096.f, AT_BELOW = 3.f;         // sum of 128 weights from which a row's reference is raised; log2 units
constexpr int AT_BOX = 128 * 64 * 2;

__device__ __forceinline__ void add2_f32(uint64_t& sum, float a, float b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum) : "l"(pack_f32x2(a, b)));
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }

template <int D, bool QS>
struct AtCfg {
  static constexpr int BOXES = D / 64;
  static constexpr int Q_PIECE = BOXES * AT_BOX;                 // a tile of queries
  static constexpr int Q_BYTES = Q_PIECE * (QS ? 2 : 1);
  static constexpr int KV_BYTES = BOXES * AT_BOX;
  static constexpr int FIT = (208 * 1024 - 2 * Q_BYTES) / (2 * KV_BYTES);
  static constexpr int STAGES = FIT > 4 ? 4 : FIT;
  static_assert(STAGES >= 2, "two tiles of keys and values");
  static constexpr int TILES = 2 * Q_BYTES + 2 * STAGES * KV_BYTES;
  static constexpr int BARS = 256;
  static constexpr int SMEM = TILES + BARS + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
};

// HALF: the cache's format.  QS: half queries over a bfloat16 cache.
template <int D, bool HALF, bool QS>
__global__ void __launch_bounds__(AT_THREADS, 1)
attn_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, AttnPrefixArgs a, uint32_t idesc_qk,
                      uint32_t idesc_pv) {
  using C = AtCfg<D, QS>;
  pdl_launch_dependents();
  pdl_wait();
  ApWork w = ap_work(a, a.first_block + blockIdx.x, threadIdx.x == 0);
  // Read from memory, these would be a thread's own to the compiler, and every operand of a product that depends on them a move to
  // a uniform register.
  w.rows = __shfl_sync(0xffffffffu, w.rows, 0);
  w.begin = __shfl_sync(0xffffffffu, w.begin, 0);
  w.end = __shfl_sync(0xffffffffu, w.end, 0);
  if (w.rows <= 0) return;
  extern __shared__ __align__(1024) uint8_t at_smem[];
  const uint32_t raw = smem_u32(at_smem);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* base_ptr = at_smem + (base - raw);
  const uint32_t q_smem = base, k_smem = base + 2 * C::Q_BYTES, v_smem = k_smem + C::STAGES * C::KV_BYTES, bar0 = base + C::TILES;
  const uint32_t b_kfull = bar0, b_kempty = b_kfull + 8 * C::STAGES, b_vfull = b_kempty + 8 * C::STAGES, b_vempty = b_vfull + 8 * C::STAGES,
                 b_clean = b_vempty + 8 * C::STAGES, b_s = b_clean + 8, b_p = b_s + 16, b_o = b_p + 16;
  static_assert(32 * C::STAGES + 8 + 48 <= C::BARS - 8, "barriers");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(base_ptr + C::TILES + C::BARS - 8);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const bool wide = w.rows > AT_ROWS;
  const int n_tiles = (w.end - w.begin + AT_KEYS - 1) / AT_KEYS;
  const auto tiles_of = [&](int x) { return wide ? n_tiles : (n_tiles + 1 - x) / 2; };          // key tiles of A and B
  const int left = w.end - w.begin - (n_tiles - 1) * AT_KEYS;                                   // rows of the last one
  // key and value tile j into its slots, by one thread
  const int cache_row = (w.seq * a.n_kv + w.kvh) * a.t_max + w.begin;
  auto load_tile = [&](int j, bool value) {
    const int s = j % C::STAGES;
    const uint32_t bar = (value ? b_vfull : b_kfull) + 8 * s;
    mbar_expect_tx(bar, C::KV_BYTES);
#pragma unroll
    for (int c = 0; c < C::BOXES; ++c)
      tma_load_2d((value ? v_smem : k_smem) + s * C::KV_BYTES + c * AT_BOX, value ? &tmap_v : &tmap_k, c * 64, cache_row + j * AT_KEYS, bar);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(b_kfull + 8 * s, 1);
      mbar_init(b_vfull + 8 * s, 1);
      mbar_init(b_kempty + 8 * s, wide ? 2 : 1);
      mbar_init(b_vempty + 8 * s, wide ? 2 : 1);
    }
    mbar_init(b_clean, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(b_s + 8 * x, 1);
      mbar_init(b_p + 8 * x, 128);
      mbar_init(b_o + 8 * x, 1);
    }
    mbar_fence_init();
    for (int j = 0; j < C::STAGES && j < n_tiles; ++j) {      // on their way while the queries are fetched
      load_tile(j, false);
      load_tile(j, true);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tmem_relinquish();
  }
  // queries, 16 bytes a thread: rows of 128 bytes, eight pieces exclusive-or swizzled by the row
  {
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;        // a negative scale turns the queries, so that maxima are maxima
    const int pieces = (wide ? 2 * AT_ROWS : AT_ROWS) * (D / 8);
    constexpr int AHEAD = 6;          // loads under way; one at a time they took 6.6 us of a CTA's start
#pragma unroll 1
    for (int base_i = threadIdx.x; base_i < pieces; base_i += AHEAD * AT_THREADS) {
      uint4 v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = base_i + u * AT_THREADS, r = i / (D / 8), c = i % (D / 8);
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (r < w.rows) {
          const int R = w.r0 + r;
          v[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + (size_t)(w.item0 + R / a.rep) * a.q_pitch +
                                                 (size_t)(w.kvh * a.rep + R % a.rep) * D + c * 8);
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = base_i + u * AT_THREADS, r = i / (D / 8), c = i % (D / 8), t = r & (AT_ROWS - 1);
        if (i >= pieces) break;
        v[u].x ^= flip; v[u].y ^= flip; v[u].z ^= flip; v[u].w ^= flip;
        uint8_t* dst = base_ptr + (r / AT_ROWS) * C::Q_BYTES + (c >> 3) * AT_BOX + t * 128 + (((c & 7) ^ (t & 7)) << 4);
        if constexpr (QS) {
          uint32_t in[4] = {v[u].x, v[u].y, v[u].z, v[u].w}, hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2_act(in[e], 1);
            hi[e] = pack2_bf16(f.x, f.y);
            const float2 h = unpack2_bf16(hi[e]);
            lo[e] = pack2_bf16(f.x - h.x, f.y - h.y);
          }
          *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(dst + C::Q_PIECE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        } else {
          *reinterpret_cast<uint4*>(dst) = v[u];
        }
      }
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // S_A [0, 128), S_B [128, 256), O_A [256, 256 + D), O_B

  // 12 warps start with 168 registers a thread; the four that move and issue keep 88, the eight that hold scores, weights and their
  // sums get 208 (88 + 2 * 208 = 3 * 168).
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(bar, parity))) {
          if (lane == 0) arcb_set_error(a.status, ARCB_DEV_WAIT_TIMEOUT_MMA);
          ok = false;
        }
      };
      int j = C::STAGES;
      for (; j < n_tiles; ++j) {
        const int s = j % C::STAGES;
        const uint32_t parity = ((j / C::STAGES) & 1) ^ 1;
        wait(b_kempty + 8 * s, parity);
        if (!ok) break;
        if (lane == 0) load_tile(j, false);
        wait(b_vempty + 8 * s, parity);
        if (!ok) break;
        if (lane == 0) load_tile(j, true);
      }
      if (ok && n_tiles > 0 && left < AT_KEYS) {
        // this warp has seen the slot's earlier tiles go, so that the barrier's parity can only mean this one
        const int s = (n_tiles - 1) % C::STAGES;
        if (__all_sync(0xffffffffu, mbar_wait_bounded(b_vfull + 8 * s, ((n_tiles - 1) / C::STAGES) & 1))) {
          uint8_t* v = base_ptr + 2 * C::Q_BYTES + (C::STAGES + s) * C::KV_BYTES;
#pragma unroll
          for (int c = 0; c < C::BOXES; ++c)
            for (int i = left * 8 + lane; i < AT_KEYS * 8; i += 32) *reinterpret_cast<uint4*>(v + c * AT_BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(b_clean);
        } else if (lane == 0) {
          arcb_set_error(a.status, ARCB_DEV_WAIT_TIMEOUT_TMA);
        }
      }
      if (!ok)        // gave up at tile j: the copies under way end before the CTA does
        for (int i = j - C::STAGES; i <= j && i < n_tiles; ++i) {
          mbar_wait_bounded(b_kfull + 8 * (i % C::STAGES), (i / C::STAGES) & 1);
          if (i < j) mbar_wait_bounded(b_vfull + 8 * (i % C::STAGES), (i / C::STAGES) & 1);
        }
    } else if (warp == 1) {
      // One warp issues for both chains in turn: with a warp each, their products shared the tensor core, both were through at the
      // same time, and both then met at the exponentials.
      const uint32_t el = elect_one();
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(bar, parity))) {
          if (lane == 0) arcb_set_error(a.status, code);
          ok = false;
        }
      };
      // The values of a tile and the scores of the next one are issued together, and all that either waits for is waited for ahead:
      // a wait between them lasted until the values were through (970 of 5450 cycles a tile).
      auto step = [&](int x, int i) {
        const int n_x = tiles_of(x);
        const uint32_t t_s = tmem_base + x * 128, t_o = tmem_base + 256 + x * D, q_tile = q_smem + (wide ? x * C::Q_BYTES : 0);
        auto tile = [&](int i) { return wide ? i : 2 * i + x; };
        const int j = tile(i), s = j % C::STAGES, j1 = tile(i - 1), s1 = j1 % C::STAGES;
        if (i < n_x) wait(b_kfull + 8 * s, (j / C::STAGES) & 1, ARCB_DEV_WAIT_TIMEOUT_TMA);
        if (i > 0) {
          wait(b_vfull + 8 * s1, (j1 / C::STAGES) & 1, ARCB_DEV_WAIT_TIMEOUT_TMA);
          if (j1 == n_tiles - 1 && left < AT_KEYS) wait(b_clean, 0, ARCB_DEV_WAIT_TIMEOUT_TMA);
          wait(b_p + 8 * x, (i - 1) & 1, ARCB_DEV_WAIT_TIMEOUT_ACC);
        }
        if (!ok) return;
        tc_fence_after();
        if (i > 0) {
          const uint64_t dv = umma_desc_mn_sw128(v_smem + s1 * C::KV_BYTES, AT_BOX);
#pragma unroll
          for (int piece = 0; piece < 2; ++piece)
#pragma unroll
            for (int ks = 0; ks < AT_KEYS / 16; ++ks)
              umma_f16_ts_if(el, t_o, t_s + piece * 64 + ks * 8, dv + (uint64_t)(ks * (2048 >> 4)), idesc_pv, (i > 1 || piece || ks) ? 1u : 0u);
        }
        if (i < n_x) {
#pragma unroll
          for (int piece = 0; piece < (QS ? 2 : 1); ++piece)
#pragma unroll
            for (int c = 0; c < C::BOXES; ++c) {
              const uint64_t dq = umma_desc_k_sw128(q_tile + piece * C::Q_PIECE + c * AT_BOX);
              const uint64_t dk = umma_desc_k_sw128(k_smem + s * C::KV_BYTES + c * AT_BOX);
#pragma unroll
              for (int ks = 0; ks < 4; ++ks) umma_f16_if(el, t_s, dq + 2 * ks, dk + 2 * ks, idesc_qk, (piece | c | ks) ? 1u : 0u);
            }
          umma_commit_if(el, b_s + 8 * x);
          umma_commit_if(el, b_kempty + 8 * s);
        }
        if (i > 0) umma_commit_if(el, b_vempty + 8 * s1);
        if (i > 0 && i == n_x) umma_commit_if(el, b_o + 8 * x);
      };
      for (int i = 0; ok && i <= tiles_of(0); ++i) {
        step(0, i);
        if (ok && i <= tiles_of(1)) step(1, i);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int x = (warp - 4) >> 2, quarter = warp & 3, n_x = tiles_of(x);
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t t_s = t_lane + x * 128, t_o = t_lane + 256 + x * D;
    constexpr float BELOW = HALF ? AT_BELOW : 0.f, RAISE = HALF ? AT_RAISE * 8.f : AT_RAISE;
    const float sc = fabsf(a.scale) * AP_LOG2E;
    const uint64_t sc2 = pack_f32x2(sc, sc);
    const int first_row = (wide ? x * AT_ROWS : 0) + quarter * 32;         // of the warp, among the CTA's
    const bool idle = first_row >= w.rows;
    bool ok = true;
    float m_ref = -INFINITY, l = 0.f;
    // 32 of the row's scores have come: hidden keys become -inf, whose exp2 is exactly 0
    auto arrived = [&](int c, int seen, uint32_t (&sv)[32]) {
      tmem_wait_ld_dep(sv);
      if (seen < AT_KEYS) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (c * 32 + e >= seen) sv[e] = 0xff800000u;
      }
    };
    auto largest = [&](int seen) {
      float mx = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t sv[32];
        tmem_ld_32x32(t_s + c * 32, sv);
        arrived(c, seen, sv);
#pragma unroll
        for (int e = 0; e < 32; e += 2) mx = max3_f32(mx, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
      }
      return fmaf(mx, sc, -BELOW);
    };
    for (int i = 0; i < n_x; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(b_s + 8 * x, i & 1))) {
        if (lane == 0) arcb_set_error(a.status, ARCB_DEV_WAIT_TIMEOUT_ACC);
        ok = false;
        break;
      }
      tc_fence_after();
      if (idle) {           // rows that do not exist: whatever their columns hold stays with them
        tc_fence_before();
        mbar_arrive(b_p + 8 * x);
        continue;
      }
      const int j = wide ? i : 2 * i + x;
      const int seen = j == n_tiles - 1 ? left : AT_KEYS;
      uint32_t pr[2][32], second[2][32];      // pairs of 64 keys each
      if (i == 0) m_ref = largest(seen);
      float total;
      // weights against the reference as it is
      auto weights = [&]() {
        const float m_safe = m_ref == -INFINITY ? 0.f : m_ref;
        const uint64_t nm2 = pack_f32x2(-m_safe, -m_safe);
        uint64_t sum[2] = {0, 0};
        uint32_t sv[2][32];
        tmem_ld_32x32(t_s, sv[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          arrived(c, seen, sv[c & 1]);
          if (c < 3) tmem_ld_32x32(t_s + (c + 1) * 32, sv[(c + 1) & 1]);      // while these are at work
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float t0, t1;
            shift2_f32(sv[c & 1][2 * e], sv[c & 1][2 * e + 1], sc2, nm2, t0, t1);
            t0 = ex2_fast(t0);
            t1 = ex2_fast(t1);
            add2_f32(sum[e & 1], t0, t1);
            const uint32_t h = pack2_prob(t0, t1, HALF ? 1 : 0);
            pr[c >> 1][(c & 1) * 16 + e] = h;
            const float2 f = unpack2_act(h, HALF ? 1 : 0);
            second[c >> 1][(c & 1) * 16 + e] = pack2_prob(t0 - f.x, t1 - f.y, HALF ? 1 : 0);
          }
        }
        float s0, s1, s2, s3;
        unpack_f32x2(sum[0], s0, s1);
        unpack_f32x2(sum[1], s2, s3);
        total = (s0 + s1) + (s2 + s3);
      };
      weights();
      // Nearly always the reference stays: maxima are looked for only where the weights' sum says that they have grown (they took a tenth
      // of the instructions).  The scores are still there.
      const bool raise = i > 0 && (total > RAISE || m_ref == -INFINITY);
      if (__any_sync(0xffffffffu, raise)) {
        const float mx = largest(seen);
        float alpha = 1.f;
        if (raise) {
          alpha = m_ref == -INFINITY ? 0.f : ex2_fast(m_ref - mx);
          m_ref = mx;
          l *= alpha;
        }
        // these scores were asked for behind the last product of values: its sums are complete
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + c * 32, o);
          tmem_wait_ld_dep(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st_32x32(t_o + c * 32, o);
        }
        weights();
      }
      l += total;
      // over scores that have all been read
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_st_32x32(t_s + c * 32, pr[c]);
        tmem_st_32x32(t_s + 64 + c * 32, second[c]);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(b_p + 8 * x);
    }
    if (!idle && ok && n_x > 0 && !__all_sync(0xffffffffu, mbar_wait_bounded(b_o + 8 * x, 0))) {
      if (lane == 0) arcb_set_error(a.status, ARCB_DEV_WAIT_TIMEOUT_ACC);
      ok = false;
    }
    const bool any = ok && n_x > 0;
    tc_fence_after();
    // With one tile of queries B's sums are handed to A's threads through the ring, which nothing reads any more.
    constexpr int REC = D + 4;
    static_assert(AT_ROWS * REC * 4 <= 2 * C::STAGES * C::KV_BYTES, "the ring holds B's sums");
    float* theirs = reinterpret_cast<float*>(base_ptr + 2 * C::Q_BYTES) + (quarter * 32 + lane) * REC;
    float fa = 1.f, fb = 0.f;
    if (!wide) {
      named_bar_sync(1, 256);
      if (x == 1 && !idle) {
        if (any)
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(t_o + c * 32, o);
            tmem_wait_ld_dep(o);
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(theirs + c * 32 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        *reinterpret_cast<float2*>(theirs + D) = any ? make_float2(m_ref, l) : make_float2(-INFINITY, 0.f);
      }
      named_bar_sync(1, 256);
      if (x == 0 && !idle) {
        const float2 ml = *reinterpret_cast<const float2*>(theirs + D);
        const float top = fmaxf(m_ref, ml.x), safe = top == -INFINITY ? 0.f : top;
        fa = exp2f(m_ref - safe);
        fb = ml.x == -INFINITY ? 0.f : exp2f(ml.x - safe);
        m_ref = top;
        l = l * fa + ml.y * fb;
      }
    }
    // results: a quad of lanes writes 64 consecutive bytes of each of its four rows
    if (!idle && (wide || x == 0)) {
      const int piece = lane & 3, quad_row = first_row + lane - piece;
      auto record = [&](int row) {
        const int R = w.r0 + row;
        return ap_record(a, (long long)(w.item0 + R / a.rep) * a.n_heads + w.kvh * a.rep + R % a.rep, w.part);
      };
      if (any) {
        const bool both = __any_sync(0xffffffffu, fb != 0.f);
        float* to[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = quad_row + e < w.rows ? record(quad_row + e) + piece * 4 : nullptr;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + c * 32, o);
          tmem_wait_ld_dep(o);
          if (both)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 v = *reinterpret_cast<const float4*>(theirs + c * 32 + e);
              o[e] = __float_as_uint(__uint_as_float(o[e]) * fa + v.x * fb);
              o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) * fa + v.y * fb);
              o[e + 2] = __float_as_uint(__uint_as_float(o[e + 2]) * fa + v.z * fb);
              o[e + 3] = __float_as_uint(__uint_as_float(o[e + 3]) * fa + v.w * fb);
            }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = make_uint4(o[g * 16 + e * 4], o[g * 16 + e * 4 + 1], o[g * 16 + e * 4 + 2], o[g * 16 + e * 4 + 3]);
            quad_transpose(v, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (to[e]) *reinterpret_cast<uint4*>(to[e] + c * 32 + g * 16) = v[e];
          }
        }
      }
      const int row = first_row + lane;
      if (row < w.rows) *reinterpret_cast<float2*>(record(row) + D) = any ? make_float2(m_ref, l) : make_float2(-INFINITY, 0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D, bool HALF, bool QS>
int at_launch(const AttnPrefixArgs& a, unsigned blocks, cudaStream_t stream) {
  using C = AtCfg<D, QS>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = arcb_opt_in_smem(attn_prefix_tc_kernel<D, HALF, QS>, C::SMEM, done);
  if (e != cudaSuccess) return (int)e;
  CUtensorMap tk, tv;
  const uint64_t rows = (uint64_t)a.n_seqs * a.n_kv * a.t_max;
  int r = arcb_make_tmap_2d_16b(&tk, a.k, rows, D, AT_KEYS, 64, HALF);
  if (!r) r = arcb_make_tmap_2d_16b(&tv, a.v, rows, D, AT_KEYS, 64, HALF);
  if (r) return 1000 + r;
  const int fmt = HALF ? 0 : 1;
  const uint32_t idesc_qk = umma_idesc_f16(AT_ROWS, AT_KEYS, fmt, fmt, 0, 0);
  const uint32_t idesc_pv = umma_idesc_f16(AT_ROWS, D, fmt, fmt, 0, 1);      // values are MN-major
  return (int)arcb_launch(attn_prefix_tc_kernel<D, HALF, QS>, dim3(blocks), dim3(AT_THREADS), C::SMEM, stream, tk, tv, a, idesc_qk, idesc_pv);
}

}  // namespace

int arcb_attn_prefix_tc(const AttnPrefixArgs& a, long long units, cudaStream_t stream) {
  if (a.kv_fmt == 1) return a.dim == 64 ? at_launch<64, true, false>(a, (unsigned)units, stream) : at_launch<128, true, false>(a, (unsigned)units, stream);
  if (a.act_fmt == 1) return a.dim == 64 ? at_launch<64, false, true>(a, (unsigned)units, stream) : -1;
  return a.dim == 64 ? at_launch<64, false, false>(a, (unsigned)units, stream) : at_launch<128, false, false>(a, (unsigned)units, stream);
}
