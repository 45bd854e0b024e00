// Attention of queries that share cached rows: arguments and launcher (attn_prefix.cu).
#pragma once
#include "common.cuh"
#include "prefix_rules.cuh"

struct AttnPrefixArgs {
  const void* q;              // item i, head h at q + i * q_pitch + h * dim (act_fmt)
  long long q_pitch;
  const void* k;              // [n_seqs][n_kv][t_max][dim] (kv_fmt)
  const void* v;
  void* out;                  // [n_items][n_heads][dim] (act_fmt)
  // group g: items [group_first[g], group_first[g + 1]) see rows [0, group_len[g]) of sequence group_seq[g].
  // uniform > 0: every group has that many items, its rows are its first item's sequence's, and group_len goes by that item.
  const int* group_first;
  const int* group_seq;
  const int* group_len;
  int uniform;
  // own rows [item_begin, item_end) of sequence item_seq (null: the item's number); item_end null: none
  const int* item_seq;
  const int* item_begin;
  const int* item_end;
  const unsigned char* item_skip;   // optional: non-zero = the row is not attended (zeros)
  int n_groups, n_items, n_heads, n_kv, dim, n_seqs, t_max;
  int max_group, max_prefix, max_own;      // what the work is planned for
  float scale;
  int act_fmt, kv_fmt;        // 0 bfloat16, 1 half, 2 fp32
  float* scratch;             // arcb_attn_prefix_scratch floats
  int* status;                // optional
  // filled by the launcher
  int rep;
  PrefixPlan plan;
  long long first_block;      // of the launch, in the numbering of the whole work
  int beside;                 // the launch runs beside the one ahead of it, whose end it waits for at its own
};

constexpr int AP_PAD = 4;     // of a partial result: the sums of a row's values, the reference of its weights (log2 units), their sum, two spare

// 16-bit formats; `a` as the launcher has filled it, units from a.first_block on.  Warps for up to 8 query rows
// (attn_prefix_rows.cu), CTAs for up to 64 (attn_prefix_mma.cu), or 256 with tcgen05 (attn_prefix_tc.cu).
int arcb_attn_prefix_rows(const AttnPrefixArgs& a, long long units, cudaStream_t stream);
int arcb_attn_prefix_mma(const AttnPrefixArgs& a, long long units, cudaStream_t stream);
int arcb_attn_prefix_tc(const AttnPrefixArgs& a, long long units, cudaStream_t stream);
// 32-bit formats, units of `tile` rows (attn_prefix_f32.cu)
int arcb_attn_prefix_f32(const AttnPrefixArgs& a, int tile, long long units, cudaStream_t stream);

bool arcb_attn_prefix_supported(int n_heads, int n_kv, int dim, int act_fmt, int kv_fmt);
// bytes of a.scratch for these sizes
long long arcb_attn_prefix_scratch(const AttnPrefixArgs& a);
int arcb_launch_attn_prefix(AttnPrefixArgs a, cudaStream_t stream);
void arcb_count_launch(long long n);
