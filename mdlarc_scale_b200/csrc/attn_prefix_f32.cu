// Attention over shared cached rows, 32-bit formats: multiply-adds.
//
// A CTA of 128 threads takes 64 cached rows at a time against up to 64 query rows, as a product of two matrices twice: every thread
// has RPT query rows x KPT keys of the scores, and of the results the same rows x D / TX columns.  Operands come from shared memory
// 16 bytes at a time, 8 x 4 of a thread's scores for 12 such loads (16 of the memory's cycles beside 128 multiply-adds a warp), so
// that the multiply-adds are what counts from 32 query rows on; below, with 4 x 2, the memory is (159 rows over 490 shared ones, 22
// groups x 32 heads of 128: 557 us, 34 TFLOP/s of the about 74 that the units have; 24 rows over 1501, 15 heads of 64: 11 us).  Tiles
// come by cp.async: the next keys while these values are at work, the next values while the next scores are.  Rows of 16-byte
// pieces are exclusive-or swizzled.  Maxima, sums and results are fp32, and so is every operand: weights are not rounded.
#include "../../include/arcb200.h"
#include "attn_prefix_impl.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"

namespace {

using namespace sm100;

constexpr int AF_KEYS = 64;

__host__ __device__ constexpr int af_smem(int rows, int dim) { return (rows * dim + 2 * AF_KEYS * dim + rows * AF_KEYS) * 4; }

// TX lanes beside each other share RPT query rows; lane tx has the keys tx, tx + TX, ...
template <int D, int TX, int RPT>
__device__ __forceinline__ void af_body(const AttnPrefixArgs& a, const ApWork& w, float* smem) {
  constexpr int ROWS = 128 / TX * RPT, KPT = AF_KEYS / TX, CPT = D / TX, VW = CPT < 4 ? CPT : 4, NV = CPT / VW, P4 = D / 4;
  float* s_q = smem;
  float* s_k = s_q + ROWS * D;
  float* s_v = s_k + AF_KEYS * D;
  float* s_p = s_v + AF_KEYS * D;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int flip = TX == 16 ? ty & 1 : 0;          // two groups of lanes in a warp read different rows: of different banks
  const size_t row0 = ((size_t)w.seq * a.n_kv + w.kvh) * (size_t)a.t_max;
  auto issue = [&](const void* from, float* to, int t, bool swizzled) {
#pragma unroll 4
    for (int i = threadIdx.x; i < AF_KEYS * P4; i += 128) {
      const int r = i / P4, c = i % P4, at = swizzled ? c ^ (r & 7) : c;
      const bool in = t + r < w.end;                // rows behind the end are zeros: a weight of 0 does not hide a NaN
      const float* src = reinterpret_cast<const float*>(from) + (row0 + (in ? t + r : w.begin)) * D + c * 4;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + r * D + at * 4)), "l"(src), "r"(in ? 16 : 0) : "memory");
    }
  };
  if (w.begin < w.end) issue(a.k, s_k, w.begin, true);
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (w.begin < w.end) issue(a.v, s_v, w.begin, false);
  asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll 4
  for (int i = threadIdx.x; i < ROWS * P4; i += 128) {
    const int r = i / P4, c = i % P4;
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < w.rows) {
      const int R = w.r0 + r;
      q = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + (size_t)(w.item0 + R / a.rep) * a.q_pitch + (size_t)(w.kvh * a.rep + R % a.rep) * D + c * 4);
    }
    *reinterpret_cast<float4*>(s_q + r * D + (TX == 16 ? c ^ (r / RPT & 1) : c) * 4) = q;
  }
  const float sc = a.scale * AP_LOG2E;
  const bool active = (int)(threadIdx.x & ~31u) / TX * RPT < w.rows;        // of the warp
  float m[RPT], l[RPT], acc[RPT][CPT];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < CPT; ++i) acc[r][i] = 0.f;
  }
  const float* q_row = s_q + ty * RPT * D;
  float* p_row = s_p + ty * RPT * AF_KEYS;
  for (int t = w.begin; t < w.end; t += AF_KEYS) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();                                // keys and queries are here
    if (active) {
      float s[RPT][KPT];
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int k = 0; k < KPT; ++k) s[r][k] = 0.f;
#pragma unroll 2
      for (int c = 0; c < P4; ++c) {
        float4 kv[KPT];
#pragma unroll
        for (int k = 0; k < KPT; ++k) kv[k] = *reinterpret_cast<const float4*>(s_k + (tx + k * TX) * D + (c ^ (tx & 7)) * 4);
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(q_row + r * D + (c ^ flip) * 4);
#pragma unroll
          for (int k = 0; k < KPT; ++k) {
            s[r][k] = fmaf(q.x, kv[k].x, s[r][k]);
            s[r][k] = fmaf(q.y, kv[k].y, s[r][k]);
            s[r][k] = fmaf(q.z, kv[k].z, s[r][k]);
            s[r][k] = fmaf(q.w, kv[k].w, s[r][k]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RPT; ++r) {
        float mx = m[r];
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
          s[r][k] = t + tx + k * TX < w.end ? s[r][k] * sc : -INFINITY;
          mx = fmaxf(mx, s[r][k]);
        }
#pragma unroll
        for (int o = TX / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float safe = mx == -INFINITY ? 0.f : mx;
        const float alpha = exp2f(m[r] - safe);
        m[r] = mx;
        l[r] *= alpha;
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
          const float p = exp2f(s[r][k] - safe);
          const int key = tx + k * TX;
          l[r] += p;
          p_row[r * AF_KEYS + (key ^ (flip << 4))] = p;
        }
#pragma unroll
        for (int i = 0; i < CPT; ++i) acc[r][i] *= alpha;
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                // values are here, keys no longer needed
    if (t + AF_KEYS < w.end) issue(a.k, s_k, t + AF_KEYS, true);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (active) {
      const int n4 = (min(AF_KEYS, w.end - t) + 3) / 4;
#pragma unroll 1
      for (int j = 0; j < n4; ++j) {
        float4 p[RPT];
#pragma unroll
        for (int r = 0; r < RPT; ++r) p[r] = *reinterpret_cast<const float4*>(p_row + r * AF_KEYS + (j ^ (flip << 2)) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v[CPT];
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const float* from = s_v + (j * 4 + e) * D + (i * TX + tx) * VW;
            if constexpr (VW == 4) *reinterpret_cast<float4*>(v + i * 4) = *reinterpret_cast<const float4*>(from);
            else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(from);
          }
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const float pe = e == 0 ? p[r].x : e == 1 ? p[r].y : e == 2 ? p[r].z : p[r].w;
#pragma unroll
            for (int i = 0; i < CPT; ++i) acc[r][i] = fmaf(pe, v[i], acc[r][i]);
          }
        }
      }
    }
    __syncthreads();                                // values no longer needed
    if (t + AF_KEYS < w.end) issue(a.v, s_v, t + AF_KEYS, false);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!active) return;
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    float sum = l[r];
#pragma unroll
    for (int o = TX / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int row = ty * RPT + r;
    if (row >= w.rows) continue;
    const int R = w.r0 + row, item = w.item0 + R / a.rep;
    const long long ih = (long long)item * a.n_heads + w.kvh * a.rep + R % a.rep;
    const bool whole = !a.plan.joined;
    float* to = whole ? reinterpret_cast<float*>(a.out) + (size_t)ih * D : ap_record(a, ih, w.part);
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const bool none = sum == 0.f || (a.item_skip && a.item_skip[item]);
#pragma unroll
      for (int i = 0; i < CPT; ++i) acc[r][i] = none ? 0.f : acc[r][i] * inv;
    } else if (tx == 0) {
      *reinterpret_cast<float2*>(to + D) = make_float2(m[r], sum);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float* at = to + (i * TX + tx) * VW;
      if constexpr (VW == 4) *reinterpret_cast<float4*>(at) = make_float4(acc[r][i * 4], acc[r][i * 4 + 1], acc[r][i * 4 + 2], acc[r][i * 4 + 3]);
      else *reinterpret_cast<float2*>(at) = make_float2(acc[r][0], acc[r][1]);
    }
  }
}

// ROWS: query rows of the largest unit
template <int D, int ROWS>
__global__ void __launch_bounds__(128, ROWS == 64 ? 2 : 4)
attn_prefix_f32_kernel(AttnPrefixArgs a) {
  pdl_launch_dependents();
  if (!a.beside) pdl_wait();
  extern __shared__ __align__(128) float af_smem_floats[];
  const ApWork w = ap_work(a, a.first_block + blockIdx.x, threadIdx.x == 0);
  if (ROWS > 32 && w.rows > 32) af_body<D, 16, 8>(a, w, af_smem_floats);
  else if (ROWS > 16 && w.rows > 16) af_body<D, 16, 4>(a, w, af_smem_floats);
  else if (w.rows > 0) af_body<D, 32, 4>(a, w, af_smem_floats);
  if (a.beside) pdl_wait();      // this launch's end is the other's too
}

// Up to R query rows: a warp a unit, without shared memory.  Eight lanes have a cached row (16 or 8 of its values each), so that a
// score takes three exchanges, and four rows are at work beside each other, each with a running maximum and sums of its own, which
// are put together at the end.  Bound by the cache's rows: 16 x 20 items of 1000 rows of 64 with 3000 shared ones, 71 us, 5.7 TB/s.  (A
// CTA of 64 keys spent its time on rows that short parts do not have: 3498 items x 32 heads of six rows at most 1.4 ms, now 0.18.)
// U: cached rows under way, of every four.
template <int D, int R, int U>
__global__ void __launch_bounds__(128, U > 1 ? 2 : R == 4 ? 3 : 4)
attn_prefix_f32_few_kernel(AttnPrefixArgs a, unsigned units) {
  pdl_launch_dependents();
  if (!a.beside) pdl_wait();
  constexpr int V4 = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 3, c = lane & 7;
  const unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  ApWork w{};
  if (unit < units) w = ap_work(a, a.first_block + unit, lane == 0);
  if (w.rows > 0) {
    float4 q[R][V4], acc[R][V4];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int R0 = w.r0 + min(r, w.rows - 1);
      const float* from = reinterpret_cast<const float*>(a.q) + (size_t)(w.item0 + R0 / a.rep) * a.q_pitch + (size_t)(w.kvh * a.rep + R0 % a.rep) * D + c * 4;
#pragma unroll
      for (int i = 0; i < V4; ++i) {
        q[r][i] = *reinterpret_cast<const float4*>(from + i * 32);
        acc[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    const float sc = a.scale * AP_LOG2E;
    const size_t row0 = (((size_t)w.seq * a.n_kv + w.kvh) * (size_t)a.t_max) * D + c * 4;
    const float* keys = reinterpret_cast<const float*>(a.k) + row0;
    const float* values = reinterpret_cast<const float*>(a.v) + row0;
    for (int t = w.begin + g; t - g < w.end; t += 4 * U) {
      float4 k[U][V4], v[U][V4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < V4; ++i) {
          const bool in = t + 4 * u < w.end;
          k[u][i] = in ? *reinterpret_cast<const float4*>(keys + (size_t)(t + 4 * u) * D + i * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[u][i] = in ? *reinterpret_cast<const float4*>(values + (size_t)(t + 4 * u) * D + i * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float s[U], mx = m[r];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[u] = 0.f;
#pragma unroll
          for (int i = 0; i < V4; ++i) {
            s[u] = fmaf(q[r][i].x, k[u][i].x, s[u]);
            s[u] = fmaf(q[r][i].y, k[u][i].y, s[u]);
            s[u] = fmaf(q[r][i].z, k[u][i].z, s[u]);
            s[u] = fmaf(q[r][i].w, k[u][i].w, s[u]);
          }
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
          s[u] = t + 4 * u < w.end ? s[u] * sc : -INFINITY;
          mx = fmaxf(mx, s[u]);
        }
        const float safe = mx == -INFINITY ? 0.f : mx, alpha = exp2f(m[r] - safe);
        m[r] = mx;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < V4; ++i) { acc[r][i].x *= alpha; acc[r][i].y *= alpha; acc[r][i].z *= alpha; acc[r][i].w *= alpha; }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float p = exp2f(s[u] - safe);
          l[r] += p;
#pragma unroll
          for (int i = 0; i < V4; ++i) {
            acc[r][i].x = fmaf(p, v[u][i].x, acc[r][i].x);
            acc[r][i].y = fmaf(p, v[u][i].y, acc[r][i].y);
            acc[r][i].z = fmaf(p, v[u][i].z, acc[r][i].z);
            acc[r][i].w = fmaf(p, v[u][i].w, acc[r][i].w);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
#pragma unroll
      for (int o = 16; o > 4; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float f = exp2f(m[r] - (top == -INFINITY ? 0.f : top));
      l[r] *= f;
#pragma unroll
      for (int o = 16; o > 4; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
      if (r >= w.rows) continue;        // of the whole warp
      const int Rr = w.r0 + r, item = w.item0 + Rr / a.rep;
      const long long ih = (long long)item * a.n_heads + w.kvh * a.rep + Rr % a.rep;
      const bool whole = !a.plan.joined, none = whole && (l[r] == 0.f || (a.item_skip && a.item_skip[item]));
      const float by = whole && !none ? 1.f / l[r] : 1.f;
      float* to = whole ? reinterpret_cast<float*>(a.out) + (size_t)ih * D : ap_record(a, ih, w.part);
#pragma unroll
      for (int i = 0; i < V4; ++i) {
        float4 o4 = make_float4(acc[r][i].x * f, acc[r][i].y * f, acc[r][i].z * f, acc[r][i].w * f);
#pragma unroll
        for (int o = 16; o > 4; o >>= 1) {
          o4.x += __shfl_xor_sync(0xffffffffu, o4.x, o);
          o4.y += __shfl_xor_sync(0xffffffffu, o4.y, o);
          o4.z += __shfl_xor_sync(0xffffffffu, o4.z, o);
          o4.w += __shfl_xor_sync(0xffffffffu, o4.w, o);
        }
        if (g == i) *reinterpret_cast<float4*>(to + i * 32 + c * 4) = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o4.x * by, o4.y * by, o4.z * by, o4.w * by);
      }
      if (!whole && lane == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top, l[r]);
    }
  }
  if (a.beside) pdl_wait();
}

template <typename... KArgs, typename... Args>
int af_start(void (*kernel)(KArgs...), const AttnPrefixArgs& a, unsigned blocks, int smem, cudaStream_t stream, Args... args) {
  return (int)(a.beside ? ap_launch_beside(kernel, dim3(blocks), dim3(128), smem, stream, a, args...)
                        : arcb_launch(kernel, dim3(blocks), dim3(128), smem, stream, a, args...));
}

template <int D, int R>
int af_few(const AttnPrefixArgs& a, unsigned units, cudaStream_t stream) {
  const unsigned blocks = (units + 3) / 4;
  // where parts are short, more warps in place of more rows under way (six at most of 3498 items x 32 heads:
  // 214 us with two, 176 with one)
  const bool brief = a.plan.shared.kernel != AP_F32_FEW && a.max_own <= 16;
  if (brief) return af_start(attn_prefix_f32_few_kernel<D, R, 1>, a, blocks, 0, stream, units);
  return af_start(attn_prefix_f32_few_kernel<D, R, (R == 4 ? 2 : 4) * (128 / D)>, a, blocks, 0, stream, units);
}

template <int D, int ROWS>
int af_tiles(const AttnPrefixArgs& a, unsigned units, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = arcb_opt_in_smem(attn_prefix_f32_kernel<D, ROWS>, af_smem(ROWS, D), done);
  return e != cudaSuccess ? (int)e : af_start(attn_prefix_f32_kernel<D, ROWS>, a, units, af_smem(ROWS, D), stream);
}

template <int D>
int af_launch(const AttnPrefixArgs& a, unsigned units, int tile, cudaStream_t stream) {
  switch (tile) {
    case 1: return af_few<D, 1>(a, units, stream);
    case 2: return af_few<D, 2>(a, units, stream);
    case 4: return af_few<D, 4>(a, units, stream);
    case 16: return af_tiles<D, 16>(a, units, stream);
    case 32: return af_tiles<D, 32>(a, units, stream);
  }
  return af_tiles<D, 64>(a, units, stream);
}

}  // namespace

int arcb_attn_prefix_f32(const AttnPrefixArgs& a, int tile, long long units, cudaStream_t stream) {
  return a.dim == 64 ? af_launch<64>(a, (unsigned)units, tile, stream) : af_launch<128>(a, (unsigned)units, tile, stream);
}
