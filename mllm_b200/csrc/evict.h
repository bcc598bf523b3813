// Host-callable launchers of the kernels that shorten requests in the paged cache: raw device pointers and a stream.
//
// Every kv head of a layer has a sum of attention weights per cached token, sums[row of the request table][kv head][cache index], in fp32.
// A request keeps the tokens with the largest sums; their cache rows, and their sums, move to the front in their order.
#pragma once

#include "kernels.h"

namespace mb200 {

// What every kernel takes of a batch.  Request b: table row req_pool_indices[b], seq_lens[b] cached tokens.
struct CacheIndex {
  const int* req_to_token;  // [table_rows, table_cols], table_stride apart; null where no slot is looked up
  const int* req_pool_indices;
  const int* seq_lens;
  int* status;
  int64_t table_stride;
  int table_rows, table_cols;   // rows and tokens that the table and the sums both have
  int batch;
};

struct WeightSums {
  float* data;              // of request row r, kv head h, token i at r * row_stride + h * head_stride + i
  int64_t row_stride, head_stride;
};

// attention of one new token per request; the weights go to the sums (weights_decode.cu)
struct WeightsDecodeArgs {
  CacheIndex index;
  WeightSums sums;
  const void* q;            // [batch, hq, head_dim], q_stride elements apart
  const void* k_cache;      // row of head h of slot s at s * kv_tok_stride + h * kv_head_stride (elements)
  const void* v_cache;
  void* out;
  float* workspace;         // weights_decode_floats()
  const float* sink;        // [hq] or null
  int64_t q_stride, out_stride, num_slots, kv_tok_stride, kv_head_stride;
  int hq, hkv, head_dim, kv_fmt, num_sms;
  float scale, logit_cap, decay;
  DType dt;
};
bool weights_decode_covers(int head_dim, int group);
int64_t weights_decode_floats(const WeightsDecodeArgs& args);
int launch_weights_decode(const WeightsDecodeArgs& args, cudaStream_t s);

// the weights that the last queries of prompts give to the cached tokens (weights_prompt.cu)
struct WeightsPromptArgs {
  CacheIndex index;
  WeightSums sums;
  const int* prefix_lens;
  const int* q_start;
  const void* q;            // [rows, hq, head_dim], q_stride elements apart
  const void* k_cache;
  float* workspace;         // weights_prompt_floats()
  const float* sink;
  int64_t q_stride, num_slots, kv_tok_stride, kv_head_stride, rows;
  int hq, hkv, head_dim, kv_fmt, num_sms, last;   // last 0: all new tokens
  bool add;
  float scale, logit_cap;
  DType dt;
};
bool weights_prompt_covers(int head_dim, int group);
int64_t weights_prompt_floats(const WeightsPromptArgs& args);
int launch_weights_prompt(const WeightsPromptArgs& args, cudaStream_t s);
int launch_weights_prompt_fp16(const WeightsPromptArgs& args, cudaStream_t s);
constexpr int kShortPromptTokens = 256;      // what the kernel for short prompts has room for (weights_prompt_short.cu)
int launch_weights_prompt_short(const WeightsPromptArgs& args, cudaStream_t s);

// which tokens stay: the last ones, the first ones, the largest sums (cache_select.cu)
struct CacheSelectArgs {
  CacheIndex index;
  const float* sums;        // [layers][rows][hkv][tokens], the strides below
  const int* budgets;       // [batch]
  int* keep;                // [layers, batch, hkv, width]
  int* counts;              // [batch]
  int64_t layer_stride, row_stride, head_stride;
  int layers, hkv, width, first, recent, pool, num_sms;
};
int launch_cache_select(const CacheSelectArgs& args, cudaStream_t s);

// cache row i <- cache row keep[i], i below counts[b], in every layer; in place (evict.cu)
struct CacheEvictArgs {
  CacheIndex index;         // without seq_lens
  void* store;              // [layers, 2, hkv, num_slots, row_bytes]
  float* sums;              // or null
  const int* keep;          // [layers, batch, hkv, width]
  const int* counts;        // [batch]
  int64_t num_slots, layer_stride, row_stride, head_stride;     // the strides are those of the sums
  int layers, hkv, width, row_bytes, num_sms;
};
int launch_cache_evict(const CacheEvictArgs& args, cudaStream_t s);

}  // namespace mb200
