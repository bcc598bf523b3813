// Host-callable launchers of the kernels for drafted token trees: raw device pointers and a stream.
//
// A batch has one tree per request.  Request b: prefix_lens[b] cached tokens and nodes j = 0 .. n - 1 (n = seq_lens[b] - prefix_lens[b]) in
// the rows q_start[b] + j and the cache slots req_to_token[req_pool_indices[b]][prefix + j]; parents[row] is a node of the same tree in
// front of the row's own, or -1.  A node's position is prefix + the number of its ancestors.
#pragma once

#include "kernels.h"

namespace mb200 {

struct TreeIndex {
  const int* req_to_token;  // [table_rows, table_cols], table_stride apart
  const int* req_pool_indices;
  const int* seq_lens;      // cached tokens and nodes
  const int* prefix_lens;
  const int* q_start;
  const int* parents;       // [rows]
  int* status;
  int64_t table_stride;
  int table_rows, table_cols, rows, batch;
};

// How the rows of a batch are laid over CTAs
struct TreePlan {
  int row_tiles, ctas, part_rows;      // row tiles side by side in a CTA; rows of a partial result
  int64_t workspace_floats;
};
TreePlan tree_plan(int head_dim, int group, int64_t rows, int64_t batch, int num_sms);

// attention of the nodes over the cached tokens, their ancestors and themselves (attention_tree.cu)
struct TreeAttnArgs {
  TreeIndex index;
  const void* q;            // [rows, hq, head_dim], q_stride elements apart
  const void* k_cache;      // row of head h of slot s at s * kv_tok_stride + h * kv_head_stride (elements)
  const void* v_cache;
  void* out;
  float* workspace;         // of the plan's size
  const float* sink;        // [hq] or null
  int64_t q_stride, out_stride, num_slots, kv_tok_stride, kv_head_stride;
  int hq, hkv, head_dim, window, chunk, kv_fmt;
  TreePlan plan;
  float scale, logit_cap;
  DType dt;
};
int launch_attention_tree(const TreeAttnArgs& args, cudaStream_t s);

// per head: norm, rotation by position * inv_freq; queries out, keys and values to the nodes' slots (tree.cu)
struct TreePrologueArgs {
  TreeIndex index;
  const void* qkv;          // [rows, hq + 2 hkv heads], qkv_stride elements apart
  const void* q_gain;       // [head_dim] or null: no norm
  const void* k_gain;
  const float* inv_freq;    // [rotated / 2], pairs (i, i + rotated / 2); rotated a multiple of 16
  const int* position_delta;   // [batch] or null
  void* q_out;              // [rows, hq, head_dim]
  void* k_cache;
  void* v_cache;
  int64_t qkv_stride, kv_tok_stride, kv_head_stride, num_slots;
  int hq, hkv, head_dim, rotated, kv_fmt;
  float eps;
  DType dt;
};
int launch_tree_prologue(const TreePrologueArgs& args, cudaStream_t s);

// cache rows of accepted nodes brought together: node i's row <- node path[i]'s, i below counts[b], in every plane of `store`
struct TreeCompactArgs {
  void* store;              // [planes, num_slots, row_bytes]
  const int* req_to_token;
  const int* req_pool_indices;
  const int* prefix_lens;
  const int* path;          // [batch, steps]
  const int* counts;        // [batch]
  int* status;
  int64_t table_stride, num_slots;
  int batch, steps, table_rows, table_cols, planes, row_bytes;
};
int launch_tree_compact(const TreeCompactArgs& args, cudaStream_t s);

// walks each request's tree with the target's filtered distribution (tree_sample.cu)
struct TreeSampleArgs {
  const void* logits;       // [rows, vocab], logit_stride elements apart, of type dt
  const int64_t* tokens;    // [rows]
  const int* parents;       // [rows]
  const int* tree_lens;     // [batch]
  const int* q_start;       // [batch]
  const float* temperature; // [batch]
  const int* top_k;         // [batch], <= 0 or >= vocab: off
  const float* top_p;       // [batch], >= 1: off
  const float* min_p;       // [batch] or null
  const float* uniform;     // [rows]
  const float* uniform_final;   // [batch]
  const float* draft;       // [rows, vocab], draft_stride apart, or null
  int* path;                // [batch, steps]
  int64_t* out;             // [batch, steps]
  int* counts;              // [batch]
  int* status;
  int64_t logit_stride, draft_stride;
  int rows, batch, vocab, steps, num_sms;
  DType dt;
};
int tree_sample_max_vocab(DType dt);
int launch_tree_sample(const TreeSampleArgs& args, cudaStream_t s);

}  // namespace mb200
