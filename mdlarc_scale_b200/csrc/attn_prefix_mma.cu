// Attention over shared cached rows in 16-bit formats: a CTA goes through a range of cached rows once for up to 64 query rows.
//
// Four warps share tiles of 64 keys and values, copied asynchronously into a ring in shared memory (16-byte pieces, exclusive-or
// swizzled by the row, so that the eight rows of a matrix load fall into different banks).  S = Q K^T and O += P V are
// m16n8k16 products with fp32 sums; queries, sums and weights stay in registers (the sums of two neighbouring score tiles are
// the weights' operand as they lie).  With 16, 32 or 64 query rows the warps divide the tile's keys among 4, 2 or 1 groups and
// the rows among 1, 2 or 4; groups are merged once at the end.  What bounds it is reading the cache with up to 16 query rows: they cost
// 16 keys x 128 dims x 3 products of 128 cycles beside 8 KB that an SM receives in 190; 16 over 7500, 20 heads of 64: 19 us with the own
// rows running beside it.  From 17 on products count, those of padding to 32 or 64 rows among them: 20 query rows over 4096 cached
// rows, 24 sequences x 8 key heads of 128 (267 MB): 79 us with the start, own rows and join, 3.4 TB/s.
//
// Rounding: weights enter the product as two 16-bit pieces (p = hi + lo, half a step of the type squared of p off).  One piece is half
// a step of a weight off, which adds up to half a step of sum p |v|: more than the output's own rounding without limit where
// values cancel, and 1.4 times its error on random ones; it took 70 us in place of the 79 above.  Half queries over a bfloat16 cache
// are two bfloat16 pieces, which is exact.  Maxima, sums and all partial results are fp32.  A range's reference is raised only when
// its maximum grows by 2^8; in half it is 2^7 below the maximum, so that weights are up to 2^15 and end at 2^-24 of it: weights down
// to 2^-32 of a range's largest one count.
#include <type_traits>

#include "attn_prefix_frag.cuh"
#include "flash_common.cuh"
#include "launch.cuh"

namespace {

constexpr int AM_KEYS = 64;
constexpr float AM_RESCALE = 8.f, AM_BELOW = 7.f;      // log2 units

template <int D>
struct AmCfg {
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int PLANE = AM_KEYS * D * 2;
  static constexpr int STAGE = 2 * PLANE;
  static constexpr int SMEM = STAGES * STAGE;
  static constexpr int MIN_CTAS = D == 64 ? 3 : 2;
};

// KG groups of keys, 4 / KG groups of 16 query rows.  HALF: the cache's format; QS: half queries over a bfloat16 cache.
template <int D, bool HALF, bool QS, int KG>
__device__ __forceinline__ void am_body(const AttnPrefixArgs& a, const ApWork& w, uint8_t* smem) {
  using C = AmCfg<D>;
  constexpr int RG = 4 / KG;
  constexpr float BELOW = HALF ? AM_BELOW : 0.f;
  constexpr int KW = AM_KEYS / KG;         // keys of a tile that a warp has
  constexpr int NT = KW / 8, DK = D / 16, CH = D / 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rg = warp / KG, kg = warp % KG;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));

  // rows of 16-byte pieces: a thread copies piece c of rows r, r + 128 / CH, ...
  const size_t row0 = ((size_t)w.seq * a.n_kv + w.kvh) * (size_t)a.t_max;
  const int c_col = threadIdx.x % CH, c_row = threadIdx.x / CH;
  const char* Kp = reinterpret_cast<const char*>(a.k) + (row0 * CH + c_col) * 16;
  const char* Vp = reinterpret_cast<const char*>(a.v) + (row0 * CH + c_col) * 16;
  auto issue = [&](int t, int stage) {
    const uint32_t st = ring + stage * C::STAGE;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane)
#pragma unroll
      for (int i = 0; i < AM_KEYS * CH / 128; ++i) {
        const int r = c_row + i * (128 / CH);
        const bool ok = t + r < w.end;
        const char* src = (plane ? Vp : Kp) + (size_t)(ok ? t + r : w.begin) * (CH * 16);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(st + plane * C::PLANE + r * (CH * 16) + ((c_col ^ (r & 7)) << 4)), "l"(src),
                     "r"(ok ? 16 : 0) : "memory");
      }
  };
  const int n_tiles = (w.end - w.begin + AM_KEYS - 1) / AM_KEYS;
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    if (i < n_tiles) issue(w.begin + i * AM_KEYS, i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // queries: row lane / 4 and that plus 8 of the warp's 16, dims (lane % 4) * 2 and that plus 8 of every 16
  const float sc = fabsf(a.scale) * AP_LOG2E;
  uint32_t q[DK][4], ql[QS ? DK : 1][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = rg * 16 + (lane >> 2) + 8 * x, R = w.r0 + r;
    const bool in = r < w.rows;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (in ? (size_t)(w.item0 + R / a.rep) * a.q_pitch + (size_t)(w.kvh * a.rep + R % a.rep) * D : 0) + (lane & 3) * 2;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;        // a negative scale turns the queries, so that maxima are maxima
#pragma unroll
    for (int ks = 0; ks < DK; ++ks)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t raw = in ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + y * 8) ^ flip : 0u;
        if constexpr (QS) {
          const float2 f = unpack2_act(raw, 1);
          am_split<false>(f.x, f.y, q[ks][2 * y + x], ql[ks][2 * y + x]);
        } else {
          q[ks][2 * y + x] = raw;
        }
      }
  }

  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const bool idle = rg * 16 >= w.rows;      // its query rows do not exist

  int get = 0, put = C::STAGES - 1;
  for (int t = 0; t < n_tiles; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncthreads();                        // the tile is here for everybody, and everybody is done with the one before
    if (t + C::STAGES - 1 < n_tiles) issue(w.begin + (t + C::STAGES - 1) * AM_KEYS, put);
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + 1 == C::STAGES ? 0 : put + 1;
    const uint32_t kst = ring + get * C::STAGE, vst = kst + C::PLANE;
    get = get + 1 == C::STAGES ? 0 : get + 1;
    const int key0 = w.begin + t * AM_KEYS + kg * KW;
    if (idle || key0 >= w.end) continue;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DK; ++ks)
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        const int r = kg * KW + n * 8 + (lane & 7) + ((lane >> 4) << 3);
        uint32_t b[4];
        am_ld4(kst + r * (CH * 16) + (((2 * ks + ((lane >> 3) & 1)) ^ (r & 7)) << 4), b);
        am_mma<HALF>(s[n], q[ks], b[0], b[1]);
        am_mma<HALF>(s[n + 1], q[ks], b[2], b[3]);
        if constexpr (QS) {
          am_mma<HALF>(s[n], ql[ks], b[0], b[1]);
          am_mma<HALF>(s[n + 1], ql[ks], b[2], b[3]);
        }
      }
    const bool part = key0 + KW > w.end;    // of the last tile: keys behind the end
    if (part)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key0 + n * 8 + (lane & 3) * 2 + (j & 1) >= w.end) s[n][j] = -INFINITY;
    float safe[2];
    bool raise = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float mx = fmaxf(s[0][2 * x], s[0][2 * x + 1]);
#pragma unroll
      for (int n = 1; n < NT; ++n) mx = max3_f32(mx, s[n][2 * x], s[n][2 * x + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = mx == -INFINITY ? -INFINITY : fmaf(mx, sc, -BELOW);
      if (mx > m[x] + AM_RESCALE || (m[x] == -INFINITY && mx > -INFINITY)) {
        const float alpha = m[x] == -INFINITY ? 0.f : ex2_fast(m[x] - mx);
        raise = true;
        safe[x] = alpha;
        m[x] = mx;
      } else {
        safe[x] = 1.f;
      }
    }
    if (__any_sync(0xffffffffu, raise)) {
      l[0] *= safe[0];
      l[1] *= safe[1];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        acc[i][0] *= safe[0]; acc[i][1] *= safe[0];
        acc[i][2] *= safe[1]; acc[i][3] *= safe[1];
      }
    }
    safe[0] = m[0] == -INFINITY ? 0.f : m[0];
    safe[1] = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float p = ex2_fast(fmaf(s[n][j], sc, -safe[j >> 1]));
        if (part && key0 + n * 8 + (lane & 3) * 2 + (j & 1) >= w.end) p = 0.f;     // also where the scale is 0
        l[j >> 1] += p;
        s[n][j] = p;
      }
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) am_split<HALF>(s[2 * kk + (y >> 1)][2 * (y & 1)], s[2 * kk + (y >> 1)][2 * (y & 1) + 1], hi[y], lo[y]);
      const int r = kg * KW + kk * 16 + (lane & 15);
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

  // the warps' results side by side in shared memory, then every query row merged over its groups of keys, in order
  constexpr int REC = D + 4;
  static_assert(4 * 16 * REC * 4 <= C::SMEM, "the results reuse the ring");
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* mine = reinterpret_cast<float*>(smem) + warp * 16 * REC;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    float* rec = mine + ((lane >> 2) + 8 * x) * REC;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(rec + i * 8 + (lane & 3) * 2) = make_float2(acc[i][2 * x], acc[i][2 * x + 1]);
    if ((lane & 3) == 0) *reinterpret_cast<float2*>(rec + D) = make_float2(m[x], l[x]);
  }
  __syncthreads();
  const bool whole = !a.plan.joined;
  for (int i = threadIdx.x; i < RG * 16 * (D / 4); i += 128) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    if (r >= w.rows) break;
    const float* rec = reinterpret_cast<const float*>(smem) + ((r >> 4) * KG * 16 + (r & 15)) * REC;
    float mt = rec[D], lt = rec[D + 1];
    float4 o = *reinterpret_cast<const float4*>(rec + c);
    if constexpr (KG > 1) {
#pragma unroll
      for (int g = 1; g < KG; ++g) mt = fmaxf(mt, rec[g * 16 * REC + D]);
      const float ms = mt == -INFINITY ? 0.f : mt;
      const float f = exp2f(rec[D] - ms);
      lt *= f;
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
      for (int g = 1; g < KG; ++g) {
        const float* other = rec + g * 16 * REC;
        const float fg = exp2f(other[D] - ms);
        const float4 v = *reinterpret_cast<const float4*>(other + c);
        lt += other[D + 1] * fg;
        o.x += v.x * fg; o.y += v.y * fg; o.z += v.z * fg; o.w += v.w * fg;
      }
    }
    const int R = w.r0 + r, item = w.item0 + R / a.rep;
    const long long ih = (long long)item * a.n_heads + w.kvh * a.rep + R % a.rep;
    if (whole) {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      o = a.item_skip && a.item_skip[item] ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      ap_store4(a.out, (size_t)ih * D + c, o, a.act_fmt);
    } else {
      float* to = ap_record(a, ih, w.part);
      *reinterpret_cast<float4*>(to + c) = o;
      if (c == 0) *reinterpret_cast<float2*>(to + D) = make_float2(mt, lt);
    }
  }
}

template <int D, bool HALF, bool QS>
__global__ void __launch_bounds__(128, AmCfg<D>::MIN_CTAS)
attn_prefix_mma_kernel(AttnPrefixArgs a) {
  pdl_launch_dependents();
  if (!a.beside) pdl_wait();
  extern __shared__ __align__(128) uint8_t am_smem[];
  const ApWork w = ap_work(a, a.first_block + blockIdx.x, threadIdx.x == 0);
  if (w.rows > 32) am_body<D, HALF, QS, 1>(a, w, am_smem);
  else if (w.rows > 16) am_body<D, HALF, QS, 2>(a, w, am_smem);
  else if (w.rows > 0) am_body<D, HALF, QS, 4>(a, w, am_smem);
  if (a.beside) pdl_wait();      // this launch's end is the other's too
}

template <int D, bool HALF, bool QS>
int am_launch(const AttnPrefixArgs& a, unsigned blocks, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = arcb_opt_in_smem(attn_prefix_mma_kernel<D, HALF, QS>, AmCfg<D>::SMEM, done);
  if (e != cudaSuccess) return (int)e;
  return (int)(a.beside ? ap_launch_beside(attn_prefix_mma_kernel<D, HALF, QS>, dim3(blocks), dim3(128), AmCfg<D>::SMEM, stream, a)
                        : arcb_launch(attn_prefix_mma_kernel<D, HALF, QS>, dim3(blocks), dim3(128), AmCfg<D>::SMEM, stream, a));
}

}  // namespace

int arcb_attn_prefix_mma(const AttnPrefixArgs& a, long long units, cudaStream_t stream) {
  if (a.kv_fmt == 1) return a.dim == 64 ? am_launch<64, true, false>(a, (unsigned)units, stream) : am_launch<128, true, false>(a, (unsigned)units, stream);
  if (a.act_fmt == 1) return a.dim == 64 ? am_launch<64, false, true>(a, (unsigned)units, stream) : am_launch<128, false, true>(a, (unsigned)units, stream);
  return a.dim == 64 ? am_launch<64, false, false>(a, (unsigned)units, stream) : am_launch<128, false, false>(a, (unsigned)units, stream);
}
