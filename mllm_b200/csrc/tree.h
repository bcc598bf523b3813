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

// attention of the nodes over the cached tokens, their ancestors and themselves (attention_tree.cu)
struct TreeAttnArgs {
  TreeIndex index;
  const void* q;            // [rows, hq, head_dim], q_stride elements apart
  const void* k_cache;      // row of head h of slot s at s * kv_tok_stride + h * kv_head_stride (elements)
  const void* v_cache;
  void* out;
  float* workspace;         // tree_workspace_floats
  const float* sink;        // [hq] or null
  int64_t q_stride, out_stride, num_slots, kv_tok_stride, kv_head_stride;
  int hq, hkv, head_dim, window, chunk, kv_fmt, ctas;
  float scale, logit_cap;
  DType dt;
};
int tree_ctas(int head_dim, int num_sms);
int64_t tree_workspace_floats(int head_dim, int group, int64_t rows, int ctas);
int launch_attention_tree(const TreeAttnArgs& args, cudaStream_t s);

}  // namespace mb200
