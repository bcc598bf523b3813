// The attention weights that the last queries of prompts give to the cached tokens, added up per token and kv head.
//
// Request b has seq_lens[b] tokens in the cache, the last n = seq - prefix of them new, with queries in rows q_start[b] + j of q.  The last
// `last` of them (all, where it is 0 or more than n) are observed: query j sees the tokens i <= place_j = prefix + j, and
//   sums_i <- (add and i < prefix: sums_i +) sum_{observed j, place_j >= i} sum_h 2^(s_hji log2 e - lse_hj)   over the heads h of the group,
// s = scale q . k (soft cap: c tanh(s / c)).  A sink is one more term of a row's normaliser, without a value.
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"

namespace mb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;

struct PromptParams {
  CacheIndex ix;
  WeightSums sums;
  const int* prefix_lens;
  const int* q_start;
  const void* q;
  const void* k_cache;
  float* lse;        // [rows][hq]
  const float* sink;
  int64_t q_stride, num_slots, kv_tok_stride, kv_head_stride;
  int rows, hkv, group, last;
  bool add;
  float scale_log2, cap_pre, cap_post;
};

struct Observed {
  int len, row, prefix, first, look;      // tokens; row of the table; cached before; row of q of the first observed query; observed ones
  bool bad;
};
__device__ __forceinline__ Observed observed_of(const PromptParams& p, int b) {
  const Cached c = cached_of(p.ix, b);
  Observed o;
  o.len = c.len;
  o.row = c.row;
  o.bad = c.bad;
  o.prefix = __ldcg(p.prefix_lens + b);
  const int start = __ldcg(p.q_start + b), n = c.len - o.prefix;
  o.look = c.len > 0 && n > 0 ? (p.last > 0 ? min(p.last, n) : n) : 0;
  if (o.look > 0 && (o.prefix < 0 || start < 0 || n > p.rows - start)) {
    o.bad = true;
    o.look = 0;
  }
  o.first = start + n - o.look;
  return o;
}

// score of one query head and one cached row, log2 domain; the query in shared memory
template <typename T, int FMT>
__device__ __forceinline__ float score(const PromptParams& p, const float* q, int head_dim, int slot, int hk) {
  if (slot < 0 || slot >= p.num_slots) return -INFINITY;
  const int64_t at = slot * p.kv_tok_stride + hk * p.kv_head_stride;
  float s = 0.f;
  for (int d = 0; d < head_dim; d += 8) {
    if constexpr (FMT == kKvSame) {
      const T* k = static_cast<const T*>(p.k_cache) + at + d;
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(q[d + i], to_f32(k[i]), s);
    } else {
      const uint8_t* k = static_cast<const uint8_t*>(p.k_cache) + at + d;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 x = unpack_fp8x2(*reinterpret_cast<const uint16_t*>(k + i), FMT);
        s = fmaf(q[d + i + 1], x.y, fmaf(q[d + i], x.x, s));
      }
    }
  }
  return p.cap_post > 0.f ? p.cap_post * tanhf(s * p.cap_pre) : s * p.scale_log2;
}

// normaliser of every observed row: a block per row and query head
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) prompt_lse_kernel(const PromptParams p, int head_dim) {
  __shared__ float q[256], red[kThreads / 32], red_sum[kThreads / 32];
  pdl_wait();
  const int t = blockIdx.x, head = blockIdx.y, hk = head / p.group;
  int place = -1, row = 0;
  for (int b = 0; b < p.ix.batch; ++b) {
    const Observed o = observed_of(p, b);
    if (o.bad && t == 0 && head == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    if (t >= o.first && t < o.first + o.look) {
      place = o.len - o.look + t - o.first;
      row = o.row;
    }
  }
  if (place < 0) return;
  for (int d = threadIdx.x; d < head_dim; d += kThreads)
    q[d] = to_f32(static_cast<const T*>(p.q)[t * p.q_stride + static_cast<int64_t>(head) * head_dim + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f;
  const int* rtt = p.ix.req_to_token + static_cast<int64_t>(row) * p.ix.table_stride;
  for (int i = threadIdx.x; i <= place; i += kThreads) {
    const int slot = rtt[i];
    if ((slot < 0 || slot >= p.num_slots) && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    const float s = score<T, FMT>(p, q, head_dim, slot, hk);
    if (s == -INFINITY) continue;
    if (s > m) {
      l *= exp2f(m - s);
      m = s;
    }
    l += exp2f(s - m);
  }
  const float top = warp_max(m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  float all = red[0];
  for (int w = 1; w < kThreads / 32; ++w) all = fmaxf(all, red[w]);
  const bool none = all == -INFINITY;
  if (p.sink != nullptr) all = fmaxf(all, p.sink[head] * kLog2e);
  const float part = warp_sum(l == 0.f ? 0.f : l * exp2f(m - all));
  if ((threadIdx.x & 31) == 0) red_sum[threadIdx.x >> 5] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = p.sink != nullptr ? exp2f(p.sink[head] * kLog2e - all) : 0.f;
    for (int w = 0; w < kThreads / 32; ++w) sum += red_sum[w];
    p.lse[static_cast<int64_t>(t) * p.hkv * p.group + head] = none ? -INFINITY : all + log2f(sum);
  }
}

// a thread per cached token; a block's tokens meet all observed rows that see them
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) prompt_sums_kernel(const PromptParams p, int head_dim) {
  __shared__ float q[256];
  pdl_wait();
  const int b = blockIdx.y, hk = blockIdx.z, i = blockIdx.x * kThreads + threadIdx.x;
  const Observed o = observed_of(p, b);
  if (o.look == 0 || static_cast<int>(blockIdx.x) * kThreads >= o.len) return;
  const int slot = i < o.len ? p.ix.req_to_token[static_cast<int64_t>(o.row) * p.ix.table_stride + i] : -1;
  float w = 0.f;
  for (int j = 0; j < o.look; ++j) {
    const int place = o.len - o.look + j;
    if (place < static_cast<int>(blockIdx.x) * kThreads) continue;
    for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
      __syncthreads();
      for (int d = threadIdx.x; d < head_dim; d += kThreads)
        q[d] = to_f32(static_cast<const T*>(p.q)[(o.first + j) * p.q_stride + static_cast<int64_t>(h) * head_dim + d]);
      __syncthreads();
      const float lse = p.lse[static_cast<int64_t>(o.first + j) * p.hkv * p.group + h];
      if (i <= place && lse != -INFINITY) w += exp2f(score<T, FMT>(p, q, head_dim, slot, hk) - lse);
    }
  }
  if (i >= o.len) return;
  float* to = p.sums.data + o.row * p.sums.row_stride + hk * p.sums.head_stride + i;
  *to = p.add && i < o.prefix ? *to + w : w;
}

template <typename T, int FMT>
int launch_one(const PromptParams& p, int head_dim, cudaStream_t s) {
  cudaError_t err = launch_pdl(prompt_lse_kernel<T, FMT>, dim3(p.rows, p.hkv * p.group), dim3(kThreads), 0, s, p, head_dim);
  note_launch();
  if (err != cudaSuccess) return -4;
  err = launch_pdl(prompt_sums_kernel<T, FMT>, dim3((p.ix.table_cols + kThreads - 1) / kThreads, p.ix.batch, p.hkv), dim3(kThreads), 0, s, p, head_dim);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

}  // namespace

bool weights_prompt_covers(int head_dim, int group) { return (head_dim == 64 || head_dim == 128 || head_dim == 256) && group >= 1 && group <= 32; }

int64_t weights_prompt_floats(const WeightsPromptArgs& a) { return a.rows * a.hq; }

int launch_weights_prompt(const WeightsPromptArgs& a, cudaStream_t s) {
  if (a.hkv <= 0 || a.hq % a.hkv != 0 || !weights_prompt_covers(a.head_dim, a.hq / a.hkv)) return -1;
  if (a.index.batch <= 0 || a.rows <= 0) return 0;
  PromptParams p{};
  p.ix = a.index;
  p.sums = a.sums;
  p.prefix_lens = a.prefix_lens;
  p.q_start = a.q_start;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.lse = a.workspace;
  p.sink = a.sink;
  p.q_stride = a.q_stride;
  p.num_slots = a.num_slots;
  p.kv_tok_stride = a.kv_tok_stride;
  p.kv_head_stride = a.kv_head_stride;
  p.rows = static_cast<int>(a.rows);
  p.hkv = a.hkv;
  p.group = a.hq / a.hkv;
  p.last = a.last;
  p.add = a.add;
  p.scale_log2 = a.scale * kLog2e;
  if (a.logit_cap > 0.f) {
    p.cap_pre = a.scale / a.logit_cap;
    p.cap_post = a.logit_cap * kLog2e;
  }
  int rc = -1;
  MB200_DISPATCH_HALF(a.dt, rc = a.kv_fmt == kKvSame ? launch_one<T, kKvSame>(p, a.head_dim, s) : a.kv_fmt == kKvE4M3 ? launch_one<T, kKvE4M3>(p, a.head_dim, s)
                                                                                                                        : launch_one<T, kKvE5M2>(p, a.head_dim, s));
  return rc;
}

}  // namespace mb200
