// What the kernels of attention over shared cached rows have in common: how a CTA finds its part of the work, where partial
// results go, how outputs are rounded.
#pragma once
#include "attn_prefix.cuh"
#include "launch.cuh"

namespace {

constexpr float AP_LOG2E = 1.4426950408889634f;
constexpr int AP_LOOK_BACK = 4096;      // groups whose ends a bad one looks at

// Launch with the programmatic attribute: the kernel's CTAs may come when all of the kernel ahead have started.
template <typename... KArgs, typename... Args>
inline cudaError_t ap_launch_beside(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}

// A CTA's part of the work: query rows (row r is item item0 + (r0 + r) / rep, head kvh * rep + (r0 + r) % rep), cached rows
// [begin, end) of a sequence, and which part of the results it is.  behind: items of a bad group that the plan has no units for.
struct ApWork {
  int item0, r0, rows, kvh, seq, begin, end, part, behind;
};

__device__ __forceinline__ float* ap_record(const AttnPrefixArgs& a, long long ih, int part) {
  return a.scratch + ((size_t)ih * a.plan.parts + part) * (a.dim + AP_PAD);
}

// Outputs saturate in half, as all of the library's do; NaN stays NaN.
__device__ __forceinline__ void ap_store4(void* out, size_t at, float4 v, int fmt) {
  if (fmt != 1 || !(isnan(v.x) || isnan(v.y) || isnan(v.z) || isnan(v.w))) {
    st_act4(out, at, v, fmt);
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
  for (int i = 0; i < 4; ++i) reinterpret_cast<__half*>(out)[at + i] = isnan(f[i]) ? __float2half_rn(f[i]) : __float2half_rn(fminf(fmaxf(f[i], -65504.f), 65504.f));
}

__device__ __forceinline__ void ap_store1(void* out, size_t at, float v, int fmt) {
  if (fmt == 1 && isnan(v)) reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
  else st_act(out, at, v, fmt);
}

// Part `part` of some items and a key head's heads when they see no rows: an empty one, or zeros where parts are not joined.  (The CTA of
// a group joins its own.)
__device__ __forceinline__ void ap_empty(const AttnPrefixArgs& a, int item0, int items, int kvh, int part) {
  for (int i = 0; i < items; ++i)
    for (int h = 0; h < a.rep; ++h) {
      const long long ih = (long long)(item0 + i) * a.n_heads + kvh * a.rep + h;
      if (a.plan.joined) *reinterpret_cast<float2*>(ap_record(a, ih, part) + a.dim) = make_float2(-INFINITY, 0.f);
      else if (!a.plan.grouped)
        for (int c = 0; c < a.dim; c += 4) ap_store4(a.out, (size_t)ih * a.dim + c, make_float4(0.f, 0.f, 0.f, 0.f), a.act_fmt);
    }
}

// Numbers: tiles of one (group, head, range) follow each other, so that they find its rows in L2.
__device__ __forceinline__ ApWork ap_work(const AttnPrefixArgs& a, long long block, bool report) {
  ApWork k;
  unsigned w = (unsigned)block;       // fewer than 2^31 (the launcher's check)
  const unsigned n1 = (unsigned)a.plan.shared.units;
  int len, at0, split, splits, grain = 15;
  if (w < n1) {
    const int t = (int)(w % a.plan.shared.tiles); w /= a.plan.shared.tiles;
    splits = a.plan.shared.splits;
    split = (int)(w % splits); w /= splits;
    k.kvh = (int)(w % a.n_kv);
    const int g = (int)(w / a.n_kv);
    int first, last;
    if (a.uniform > 0) {
      first = g * a.uniform;
      last = first + a.uniform;
      k.seq = first;
      len = a.group_len[first];
    } else {
      first = a.group_first[g];
      last = a.group_first[g + 1];
      k.seq = a.group_seq[g];
      len = a.group_len[g];
    }
    const bool bad = first < 0 || last < first || last > a.n_items || last - first > a.max_group || len < 0 || len > a.t_max ||
                     (len > 0 && (k.seq < 0 || k.seq >= a.n_seqs)) || (g == 0 && first != 0) || (g == a.n_groups - 1 && last != a.n_items);
    k.behind = 0;
    if (bad) {
      // Its items see no shared rows.  They begin at the largest end of the groups ahead of it and end at its own, n_items if it is the last
      // group; ends outside the items count for nothing.  So no item is left out, whatever the ends are: going from group to group, the
      // largest end so far rises from 0 to n_items.  One that is further back than the loop goes only makes an item a bad group's too.
      if (report) arcb_set_error(a.status, ARCB_DEV_BAD_INDEX);
      if (a.uniform <= 0) {
        if (g == a.n_groups - 1) last = a.n_items;
        first = 0;
        if (last >= 0 && last <= a.n_items) {
          for (int i = max(1, g - AP_LOOK_BACK); i <= g; ++i) {
            const int end = a.group_first[i];
            if (end <= a.n_items) first = max(first, end);
          }
        }
        if (last < first || last > a.n_items) last = first;
      }
      len = 0;
      if (last - first > a.max_group) {
        k.behind = last - first - a.max_group;
        last = first + a.max_group;
        if (report && t == 0) ap_empty(a, last, k.behind, k.kvh, split);
      }
    }
    k.item0 = first;
    k.r0 = t * a.plan.shared.tile;
    k.rows = min(a.plan.shared.tile, (last - first) * a.rep - k.r0);
    at0 = 0;
    grain = a.plan.shared.kernel == AP_TC ? 127 : a.plan.shared.kernel == AP_ROWS ? 15 : 63;
    k.part = split;
  } else {
    w -= n1;
    splits = a.plan.own.splits;
    split = (int)(w % splits); w /= splits;
    const int t = (int)(w % a.plan.own.tiles); w /= a.plan.own.tiles;
    k.kvh = (int)(w % a.n_kv);
    k.item0 = (int)(w / a.n_kv);
    k.r0 = t * a.plan.own.tile;
    k.rows = min(a.plan.own.tile, a.rep - k.r0);
    k.seq = a.item_seq ? a.item_seq[k.item0] : k.item0;
    at0 = a.item_begin ? a.item_begin[k.item0] : 0;
    len = ap_row_count(at0, a.item_end[k.item0], k.seq, a.n_seqs, a.t_max);
    if (len < 0) {
      if (report) arcb_set_error(a.status, ARCB_DEV_BAD_INDEX);
      len = 0;
    }
    if (a.item_skip && a.item_skip[k.item0]) len = 0;
    grain = a.plan.own.kernel == AP_ROWS ? 15 : 63;
    k.part = a.plan.shared.splits + split;
  }
  int chunk = (len + splits - 1) / splits;
  chunk = (chunk + grain) & ~grain;
  k.begin = at0 + min(split * chunk, len);
  k.end = at0 + min((split + 1) * chunk, len);
  return k;
}

}  // namespace
