// Attention of queries that share cached rows (samples of one prompt, requests behind one preamble, draft tokens of a
// sequence): o = softmax(scale q K^T) V over the rows of the item's group and the rows of its own.
//
// A softmax over a set of rows can be put together from parts: with m = max, l = sum exp(s - m), a = sum exp(s - m) v of every
// part, the whole is sum_i a_i exp(m_i - m) / sum_i l_i exp(m_i - m), m = max m_i.  So the shared rows are gone through once for
// all queries of a group that use a key head (items x rep rows), the own rows once an item, and a last kernel joins the parts.
#include <cmath>

#include "../../include/arcb200.h"
#include "attn_prefix_impl.cuh"
#include "gemm.cuh"
#include "launch.cuh"

int arcb_fail(int code, const char* msg);
int arcb_fail_cuda(cudaError_t e, const char* where);

namespace {

// Joins the parts of an (item, head) in order, a warp for each: the maximum of all, then their sums with lane s at the factor of
// every 32nd part.
__global__ void __launch_bounds__(128)
attn_prefix_join_kernel(AttnPrefixArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long ih = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (ih >= (long long)a.n_items * a.n_heads) return;
  const int n = a.plan.parts, rec = a.dim + AP_PAD, c = lane * 4;
  const float* r0 = a.scratch + (size_t)ih * n * rec;
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, r0[(size_t)s * rec + a.dim]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float safe = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < n; base += 32) {
    float f = 0.f;
    if (base + lane < n) {
      const float2 ml = *reinterpret_cast<const float2*>(r0 + (size_t)(base + lane) * rec + a.dim);
      f = exp2f(ml.x - safe);
      l += ml.y * f;
    }
    const int here = min(32, n - base);
#pragma unroll 8
    for (int i = 0; i < here; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      if (c < a.dim && fi != 0.f) {        // an empty part's sums count for nothing, whatever they are
        const float4 v = *reinterpret_cast<const float4*>(r0 + (size_t)(base + i) * rec + c);
        sum.x += v.x * fi; sum.y += v.y * fi; sum.z += v.z * fi; sum.w += v.w * fi;
      }
    }
  }
  l = warp_sum(l);
  if (c >= a.dim) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  sum = a.item_skip && a.item_skip[ih / a.n_heads] ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
  ap_store4(a.out, (size_t)ih * a.dim + c, sum, a.act_fmt);
}

// Few results of many parts: a CTA for each; warp j takes parts j, j + 4, ... in order, eight at a time, so that their sums and
// maxima travel together; the warps' results are joined in order.
__global__ void __launch_bounds__(128)
attn_prefix_join_cta_kernel(AttnPrefixArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int AHEAD = 8, W = 4;
  __shared__ float4 s_sum[W][32];
  __shared__ float2 s_ml[W];
  const int lane = threadIdx.x & 31, mine = threadIdx.x >> 5;
  const long long ih = blockIdx.x;
  const int n = a.plan.parts, rec = a.dim + AP_PAD, c = min(lane * 4, a.dim - 4);
  const float* r0 = a.scratch + (size_t)ih * n * rec;
  float m = -INFINITY, l = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](const float2* ml, const float4* v, int count) {
    float top = m;
#pragma unroll
    for (int i = 0; i < count; ++i) top = fmaxf(top, ml[i].x);
    const float safe = top == -INFINITY ? 0.f : top;
    const float f0 = exp2f(m - safe);
    l *= f0;
    sum.x *= f0; sum.y *= f0; sum.z *= f0; sum.w *= f0;
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const float f = exp2f(ml[i].x - safe);
      l += ml[i].y * f;
      if (ml[i].x != -INFINITY) {        // an empty part's sums count for nothing, whatever they are
        sum.x += v[i].x * f; sum.y += v[i].y * f; sum.z += v[i].z * f; sum.w += v[i].w * f;
      }
    }
    m = top;
  };
  for (int base = mine; base < n; base += AHEAD * W) {
    float2 ml[AHEAD];
    float4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int s = base + i * W;
      ml[i] = s < n ? *reinterpret_cast<const float2*>(r0 + (size_t)s * rec + a.dim) : make_float2(-INFINITY, 0.f);
      v[i] = s < n ? *reinterpret_cast<const float4*>(r0 + (size_t)s * rec + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    join(ml, v, AHEAD);
  }
  s_sum[mine][lane] = sum;
  if (lane == 0) s_ml[mine] = make_float2(m, l);
  __syncthreads();
  if (mine != 0) return;
  float2 ml[W - 1];
  float4 v[W - 1];
#pragma unroll
  for (int i = 1; i < W; ++i) {
    ml[i - 1] = s_ml[i];
    v[i - 1] = s_sum[i][lane];
  }
  join(ml, v, W - 1);
  if (lane * 4 >= a.dim) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  sum = a.item_skip && a.item_skip[ih / a.n_heads] ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
  ap_store4(a.out, (size_t)ih * a.dim + c, sum, a.act_fmt);
}

void fill_plan(AttnPrefixArgs& a) {
  a.rep = a.n_heads / a.n_kv;
  // tcgen05 from 640 shared rows on (64 items of 4 heads, 8 groups: 51.5 us with it and 48.2 without at 512 rows, 52.7 and 52.4 at 640, 56.1
  // and 60.8 at 768, 61.4 and 67.0 at 1024; 24 items 29.9 and 29.7 at 600, 32.4 and 37.0 at 768); half queries over bfloat16, whose scores
  // take two products, from 2048 on (128 items of 20 heads: 39.5 us and 36.8 at 1500, 41.1 and 40.9 at 2100, 44.3 and 45.1 at 3000).
  const bool split = a.act_fmt != a.kv_fmt;
  const bool tc = a.kv_fmt != 2 && (!split || a.dim == 64) && a.scale != 0.f && a.max_prefix >= (split ? 2048 : 640);
  a.plan = prefix_plan(a.n_groups, a.max_group, a.max_prefix, a.n_items, a.item_end ? a.max_own : 0, a.n_kv, a.rep, a.dim, a.kv_fmt == 2, tc, arcb_num_sms());
}

int launch_part(const AttnPrefixArgs& a, const PrefixPart& p, long long units, cudaStream_t stream) {
  arcb_count_launch(1);
  switch (p.kernel) {
    case AP_ROWS: return arcb_attn_prefix_rows(a, units, stream);
    case AP_TILES: return arcb_attn_prefix_mma(a, units, stream);
    case AP_TC: return arcb_attn_prefix_tc(a, units, stream);
  }
  return arcb_attn_prefix_f32(a, p.tile, units, stream);
}

}  // namespace

bool arcb_attn_prefix_supported(int n_heads, int n_kv, int dim, int act_fmt, int kv_fmt) {
  return n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0 && (dim == 64 || dim == 128) &&
         (act_fmt == kv_fmt || (act_fmt == 1 && kv_fmt == 0));
}

long long arcb_attn_prefix_scratch(const AttnPrefixArgs& args) {
  AttnPrefixArgs a = args;
  fill_plan(a);
  return a.plan.joined ? (long long)a.n_items * a.n_heads * a.plan.parts * (a.dim + AP_PAD) * 4 : 0;
}

int arcb_launch_attn_prefix(AttnPrefixArgs a, cudaStream_t stream) {
  if (a.n_items <= 0) return 0;
  fill_plan(a);
  const PrefixPlan& p = a.plan;
  if (p.parts < 1 || (p.joined && !a.scratch)) return -1;
  const long long joins = ((long long)a.n_items * a.n_heads + 3) / 4;
  if (p.shared.units + p.own.units > 0x7fffffffLL || joins > 0x1fffffffLL) return -1;
  a.first_block = 0;
  a.beside = 0;
  int r = 0;
  if (p.shared.units > 0) r = launch_part(a, p.shared, p.shared.units + (p.together ? p.own.units : 0), stream);
  if (r == 0 && p.own.units > 0 && !p.together) {
    a.first_block = p.shared.units;
    // Beside the shared part, which it does not depend on.  What came before that one is over when it starts, unless the library
    // launches everything programmatically.
    a.beside = p.shared.units > 0 && !arcb_pdl_enabled();
    r = launch_part(a, p.own, p.own.units, stream);
  }
  if (r || !p.joined) return r;
  // Its CTAs come while the last ones of the parts are at work, and wait.  Four warps a result where a warp each would leave SMs without
  // work (two samples in four parts: 9.3 us in all with a warp each, 7.7 with four).
  const bool few = joins < 4LL * arcb_num_sms();
  arcb_count_launch(1);
  return (int)(few ? ap_launch_beside(attn_prefix_join_cta_kernel, dim3((unsigned)((long long)a.n_items * a.n_heads)), dim3(128), 0, stream, a)
                   : ap_launch_beside(attn_prefix_join_kernel, dim3((unsigned)joins), dim3(128), 0, stream, a));
}

static int to_fmt(int act_format) { return act_format == ARCB_ACT_F16 ? 1 : act_format == ARCB_ACT_BF16 ? 0 : 2; }

// Checks and converts; the message says what is wrong.
static int prefix_args(const arcb_prefix_attention_args* p, AttnPrefixArgs& a, bool sizes_only) {
  if (!p) return arcb_fail(ARCB_E_ARG, "null argument");
  if (p->n_items <= 0 || p->n_heads <= 0 || p->n_kv <= 0 || p->n_seqs <= 0 || p->t_max <= 0 || p->n_groups < 0)
    return arcb_fail(ARCB_E_ARG, "bad prefix attention sizes");
  if (p->n_heads % p->n_kv) return arcb_fail(ARCB_E_ARG, "n_kv must divide n_heads");
  if (p->act_format < ARCB_ACT_F16 || p->act_format > ARCB_ACT_F32 || p->kv_format < ARCB_ACT_F16 || p->kv_format > ARCB_ACT_F32)
    return arcb_fail(ARCB_E_ARG, "unknown act_format or kv_format");
  a.act_fmt = to_fmt(p->act_format);
  a.kv_fmt = to_fmt(p->kv_format);
  if (!arcb_attn_prefix_supported(p->n_heads, p->n_kv, p->dim, a.act_fmt, a.kv_fmt))
    return arcb_fail(ARCB_E_UNSUPPORTED, "prefix attention: heads of 64 or 128, queries in the cache's format or half over a bfloat16 cache");
  if (!std::isfinite(p->scale)) return arcb_fail(ARCB_E_ARG, "scale must be finite");
  a.n_groups = p->n_groups; a.n_items = p->n_items; a.n_heads = p->n_heads; a.n_kv = p->n_kv; a.dim = p->dim; a.n_seqs = p->n_seqs; a.t_max = p->t_max;
  auto bound = [](int v, int most) { return v <= 0 || v > most ? most : v; };
  a.max_group = bound(p->max_group, p->n_items);
  a.max_prefix = bound(p->max_prefix, p->t_max);
  a.max_own = bound(p->max_own, p->t_max);
  a.item_end = p->d_item_end; a.scale = p->scale;
  if (!p->n_groups && !p->d_item_end) return arcb_fail(ARCB_E_ARG, "prefix attention needs groups, rows of the items' own, or both");
  if (a.kv_fmt != 2 && (long long)p->n_seqs * p->n_kv * p->t_max >= (1ll << 31) - 256) return arcb_fail(ARCB_E_UNSUPPORTED, "prefix attention: caches of 2^31 rows");
  if (sizes_only) return ARCB_OK;
  if (!p->d_q || !p->d_k || !p->d_v || !p->d_out) return arcb_fail(ARCB_E_ARG, "null attention argument");
  if (p->n_groups && (!p->d_group_first || !p->d_group_seq || !p->d_group_len)) return arcb_fail(ARCB_E_ARG, "null group arrays");
  const long long pitch = p->q_pitch ? p->q_pitch : (long long)p->n_heads * p->dim;
  const int es = a.act_fmt == 2 ? 4 : 2;
  if (pitch < 0 || (pitch * es) % 16) return arcb_fail(ARCB_E_ARG, "q_pitch must be a multiple of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(p->d_q) | reinterpret_cast<uintptr_t>(p->d_k) | reinterpret_cast<uintptr_t>(p->d_v) |
       reinterpret_cast<uintptr_t>(p->d_out) | reinterpret_cast<uintptr_t>(p->d_scratch)) % 16)
    return arcb_fail(ARCB_E_ARG, "attention arrays must be aligned to 16 bytes");
  a.q = p->d_q; a.q_pitch = pitch; a.k = p->d_k; a.v = p->d_v; a.out = p->d_out;
  a.group_first = p->d_group_first; a.group_seq = p->d_group_seq; a.group_len = p->d_group_len;
  a.item_seq = p->d_item_seq; a.item_begin = p->d_item_begin; a.item_skip = p->d_item_skip;
  a.scratch = reinterpret_cast<float*>(p->d_scratch); a.status = p->d_status;
  return ARCB_OK;
}

extern "C" int64_t arcb_prefix_attention_scratch_bytes(const arcb_prefix_attention_args* p) {
  AttnPrefixArgs a{};
  const int r = prefix_args(p, a, true);
  return r ? r : arcb_attn_prefix_scratch(a);
}

extern "C" int arcb_op_prefix_attention(const arcb_prefix_attention_args* p, void* stream) {
  AttnPrefixArgs a{};
  const int r = prefix_args(p, a, false);
  if (r) return r;
  const long long need = arcb_attn_prefix_scratch(a);
  if (need > 0 && (!p->d_scratch || p->scratch_bytes < need))
    return arcb_fail(ARCB_E_ARG, "scratch is smaller than arcb_prefix_attention_scratch_bytes");
  const int e = arcb_launch_attn_prefix(a, (cudaStream_t)stream);
  if (e >= 1000) return arcb_fail(ARCB_E_UNSUPPORTED, "prefix attention: no tensor map for these arrays");
  if (e > 0) return arcb_fail_cuda((cudaError_t)e, "prefix attention");
  if (e < 0) return arcb_fail(ARCB_E_ARG, "prefix attention: too much work for one call");
  return ARCB_OK;
}
