// Launches on a paged K/V cache that the batched decode step (mq_prefill.hip) shares with the C
// entry points of mq_pages.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "megaqwen_amd.h"

namespace mq {
namespace pg {

struct AppendArgs {
  uint16_t *k, *v, *bounds;  // one layer of the pool; bounds may be null
  const uint16_t *kr, *vr;   // the new rows [batch, kv heads, d]
  int64_t k_sb, k_sh, v_sb, v_sh;
  const int *tables, *lens;
  int64_t t_sb;
  int num_pages, hkv, lp, d, width, batch;
};

struct AttnArgs {
  const uint16_t *k, *v;  // one layer of the pool
  const uint16_t* q;      // [batch, hq, d]
  uint16_t* out;
  int64_t q_sb, q_sh, o_sb, o_sh;
  const int *prefix_pages, *tables, *lens;
  int64_t t_sb, t_sh;  // table of (sequence, kv head)
  float* part_o;       // [np + ns, batch, hq, d] and (maximum, sum) [np + ns, batch, hq]
  float2* part_ml;
  uint32_t* tickets;  // [batch, hkv, own_tiles], zero (OWN only)
  int num_pages, hkv, hq, g, lp, width, batch;
  int prefix_len, len_add;  // len_add: rows appended since lens was written
  int prefix_tiles, np, own_tiles, groups, ns;  // groups: of sequences, one or (a wave each) four of them
  float scale_log2;
};

struct SelectArgs {
  const uint16_t *q, *bounds;
  int64_t q_sb, q_sh, t_sb;
  const int *tables, *lens;
  int *chosen, *pages, *sub_lens;  // [batch, hkv, top] logical and physical, [batch] rows in them
  uint32_t* tickets;               // [batch, hkv, own_tiles], cleared here
  int num_pages, hkv, g, lp, width, top, len_add, own_tiles;
};

// How an attention call is split: the form and number of the prefix's row tiles, parts of the
// prefix and of the own rows, and the workspace: the partial outputs, then the maxima and sums.
struct AttnPlan {
  int form, prefix_tiles, np, own_tiles, groups, ns;
  size_t out_bytes, bytes;
};
AttnPlan plan_attention(int batch, int hkv, int g, int d, int prefix_len, int max_len);

// Bytes of workspace of sparse_attention
size_t sparse_workspace(int batch, int hkv, int g, int d, int top, int width, int page_size);

// The entry points' work; len_add: rows appended since `lens` was written.
int append_rows(const AppendArgs& A, bool f16, hipStream_t stream);
int shared_attention(const MqPagePool* P, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
                     int num_q_heads, int batch, const int* prefix_pages, int prefix_len, const int* tables, int64_t t_sb,
                     int width, const int* lens, int len_add, int max_len, float scale, void* ws, size_t ws_bytes,
                     hipStream_t stream);
int sparse_attention(const MqPagePool* P, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
                     int* chosen, int num_q_heads, int batch, const int* tables, int64_t t_sb, int width, const int* lens,
                     int len_add, int top, float scale, void* ws, size_t ws_bytes, hipStream_t stream);

}  // namespace pg
}  // namespace mq
