// PyTorch binding of the kernels that shorten requests in the paged cache, part of the module of latent attention.
#pragma once

#include <algorithm>
#include <cfloat>
#include <utility>
#include <vector>

#include "bindings_common.h"
#include "bindings_tree.h"      // CHECK_ARG
#include "evict.h"

namespace {

void check_ints(const Tensor& t, int64_t n, const char* name, const Tensor& like) {
  CHECK_ARG(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1 && t.numel() == n, "mllm_b200: ", name,
            " must be a contiguous int32 vector of ", n, " elements on ", like.device());
}

mb200::CacheIndex cache_index(const char* what, const c10::optional<Tensor>& req_to_token, const Tensor& req_pool_indices,
                              const c10::optional<Tensor>& seq_lens, const c10::optional<Tensor>& sums, const Tensor& like) {
  const int64_t batch = req_pool_indices.numel();
  CHECK_ARG(batch < (int64_t(1) << 24), what, ": too many requests");
  check_ints(req_pool_indices, batch, "req_pool_indices", like);
  mb200::CacheIndex ix{};
  int64_t rows = INT32_MAX, cols = INT32_MAX;
  if (req_to_token.has_value()) {
    CHECK_ARG(req_to_token->device() == like.device() && req_to_token->dim() == 2 && req_to_token->scalar_type() == at::kInt &&
                  (req_to_token->stride(1) == 1 || req_to_token->size(1) == 1),
              what, ": req_to_token must be a two-dimensional int32 tensor with unit inner stride on ", like.device());
    ix.req_to_token = req_to_token->data_ptr<int>();
    ix.table_stride = req_to_token->stride(0);
    rows = req_to_token->size(0);
    cols = req_to_token->size(1);
  }
  if (seq_lens.has_value()) {
    check_ints(*seq_lens, batch, "seq_lens", like);
    ix.seq_lens = seq_lens->data_ptr<int>();
  }
  if (sums.has_value()) {
    rows = std::min(rows, sums->size(-3));
    cols = std::min(cols, sums->size(-1));
  }
  CHECK_ARG(rows <= INT32_MAX && cols <= INT32_MAX, what, ": too many rows or tokens");
  ix.req_pool_indices = req_pool_indices.data_ptr<int>();
  ix.status = device_state(like.get_device()).status.data_ptr<int>();
  ix.table_rows = static_cast<int>(rows);
  ix.table_cols = static_cast<int>(cols);
  ix.batch = static_cast<int>(batch);
  return ix;
}

void check_sums(const char* what, const Tensor& sums, int64_t dims, int64_t heads, const Tensor& like) {
  CHECK_ARG(sums.device() == like.device() && sums.scalar_type() == at::kFloat && sums.dim() == dims && sums.size(-2) == heads &&
                (sums.stride(-1) == 1 || sums.size(-1) == 1),
            what, ": sums must be fp32 [", dims == 4 ? "layers, " : "", "requests, ", heads, ", tokens] with unit inner stride on ", like.device());
}

// Whether no element of a tensor that is written lies where another does (an expanded tensor's do)
bool apart(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;       // stride, size
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 0) return true;
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  }
  std::sort(dims.begin(), dims.end());
  int64_t span = 1;
  for (const auto& d : dims) {
    if (d.first < span) return false;
    span += d.first * (d.second - 1);
  }
  return true;
}

void check_written_sums(const char* what, const Tensor& sums, int64_t dims, int64_t heads, const Tensor& like) {
  check_sums(what, sums, dims, heads, like);
  CHECK_ARG(apart(sums), what, ": sums are written: their rows and heads must not overlap");
}

void check_queries(const char* what, const Tensor& q, int64_t hkv) {
  CHECK_ARG(q.is_cuda() && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf), what, ": q must be a bf16 or fp16 device tensor");
  CHECK_ARG(q.dim() == 3 && q.stride(2) == 1 && q.stride(1) == q.size(2) && q.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0,
            what, ": q must be [rows, heads, features], heads of a row contiguous, rows on 16-byte boundaries");
  CHECK_ARG(hkv > 0 && q.size(1) > 0 && q.size(1) % hkv == 0, what, ": ", q.size(1), " query heads over ", hkv, " key heads");
}

// 0: the cache holds `like`'s type; 1 / 2: unscaled e4m3 / e5m2
int cache_format(const char* what, const Tensor& cache, const Tensor& like) {
  const auto ct = cache.scalar_type();
  const int fmt = ct == like.scalar_type() ? 0 : ct == at::kFloat8_e4m3fn ? 1 : ct == at::kFloat8_e5m2 ? 2 : -1;
  const int64_t unit = fmt == 0 ? 8 : 16;       // elements of 16 bytes
  CHECK_ARG(fmt >= 0 && cache.dim() == 3 && cache.size(2) == like.size(2) && cache.stride(2) == 1 && cache.stride(0) % unit == 0 &&
                cache.stride(1) % unit == 0 && cache.device() == like.device() && cache.size(0) < (int64_t(1) << 31) &&
                (reinterpret_cast<uintptr_t>(cache.data_ptr()) & 15) == 0,
            what, ": caches must be [slots, heads, features] views of the queries' type, float8_e4m3fn or float8_e5m2 on their device, with unit "
            "inner stride and rows on 16-byte boundaries");
  return fmt;
}

void check_scores(const char* what, double scale, double cap, const c10::optional<Tensor>& sink, const Tensor& q) {
  constexpr double kMost = FLT_MAX / 2;         // times log2 e it is finite still
  CHECK_ARG(scale >= FLT_MIN && scale <= kMost, what, ": scale must be positive and at most ", kMost, ", not ", scale);
  CHECK_ARG(cap == 0. || (cap >= FLT_MIN && cap <= kMost), what, ": logit_cap must be 0, or positive and at most ", kMost, ", not ", cap);
  if (sink.has_value())
    CHECK_ARG(sink->device() == q.device() && sink->scalar_type() == at::kFloat && sink->is_contiguous() && sink->dim() == 1 && sink->numel() == q.size(1),
              what, ": sink must be fp32 [", q.size(1), "] on ", q.device());
}

Tensor attention_decode_weights(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& req_to_token,
                                const Tensor& req_pool_indices, const Tensor& seq_lens, double scale, const Tensor& sums, double decay,
                                const c10::optional<Tensor>& given, double logit_cap, const c10::optional<Tensor>& sink) {
  const char* what = "attention_decode_weights";
  const int64_t hkv = k_cache.dim() == 3 ? k_cache.size(1) : 0;
  check_queries(what, q, hkv);
  mb200::WeightsDecodeArgs a{};
  a.kv_fmt = cache_format(what, k_cache, q);
  CHECK_ARG(cache_format(what, v_cache, q) == a.kv_fmt && v_cache.sizes() == k_cache.sizes() && v_cache.strides() == k_cache.strides(), what,
            ": the caches must be of one layout and type");
  const int64_t batch = req_pool_indices.numel(), hd = q.size(2);
  CHECK_ARG(q.size(0) == batch, what, ": q has ", q.size(0), " rows for ", batch, " requests");
  CHECK_ARG(mb200::weights_decode_covers(static_cast<int>(hd), static_cast<int>(q.size(1) / hkv)), what, ": ", q.size(1), " heads of ", hd,
            " features over ", hkv, " key heads: heads of 64, 128 or 256 features, groups of up to 32 heads (16 of 256 features)");
  check_written_sums(what, sums, 3, hkv, q);
  check_scores(what, scale, logit_cap, sink, q);
  CHECK_ARG(decay >= 0. && decay <= 1., what, ": decay must be from 0 to 1, not ", decay);
  Tensor out = given.has_value() ? *given : torch::empty(q.sizes(), q.options());
  CHECK_ARG(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device() && out.stride(2) == 1 &&
                out.stride(1) == hd && apart(out),
            what, ": out must be like q, heads of a row contiguous, rows apart");
  c10::cuda::CUDAGuard g(q.device());
  a.index = cache_index(what, req_to_token, req_pool_indices, seq_lens, sums, q);
  a.sums = {sums.data_ptr<float>(), sums.stride(0), sums.stride(1)};
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.out = out.data_ptr();
  a.sink = sink.has_value() ? sink->data_ptr<float>() : nullptr;
  a.q_stride = q.stride(0);
  a.out_stride = out.stride(0);
  a.num_slots = k_cache.size(0);
  a.kv_tok_stride = k_cache.stride(0);
  a.kv_head_stride = k_cache.stride(1);
  a.hq = static_cast<int>(q.size(1));
  a.hkv = static_cast<int>(hkv);
  a.head_dim = static_cast<int>(hd);
  a.num_sms = device_state(q.get_device()).num_sms;
  a.scale = static_cast<float>(scale);
  a.logit_cap = static_cast<float>(logit_cap);
  a.decay = static_cast<float>(decay);
  a.dt = dtype_of(q);
  CHECK_ARG(batch * a.hq < (int64_t(1) << 30), what, ": too many rows");
  // of this call alone: the caching allocator hands it out again in stream order, and a captured graph has its own
  Tensor ws = torch::empty({mb200::weights_decode_floats(a)}, q.options().dtype(torch::kFloat32));
  a.workspace = ws.data_ptr<float>();
  const int rc = mb200::launch_weights_decode(a, stream_of(q));
  TORCH_CHECK(rc == 0, "mllm_b200 attention_decode_weights: unsupported configuration or launch failure (code ", rc, ")");
  return out;
}

void attention_prefill_weights(const Tensor& q, const Tensor& k_cache, const Tensor& req_to_token, const Tensor& req_pool_indices,
                               const Tensor& seq_lens, const Tensor& prefix_lens, const Tensor& q_start, double scale, const Tensor& sums,
                               int64_t last, bool add, double logit_cap, const c10::optional<Tensor>& sink) {
  const char* what = "attention_prefill_weights";
  const int64_t hkv = k_cache.dim() == 3 ? k_cache.size(1) : 0;
  check_queries(what, q, hkv);
  mb200::WeightsPromptArgs a{};
  a.kv_fmt = cache_format(what, k_cache, q);
  const int64_t batch = req_pool_indices.numel(), hd = q.size(2);
  CHECK_ARG(mb200::weights_prompt_covers(static_cast<int>(hd), static_cast<int>(q.size(1) / hkv)), what, ": ", q.size(1), " heads of ", hd,
            " features over ", hkv, " key heads: heads of 64, 128 or 256 features, groups of up to 32 heads");
  check_written_sums(what, sums, 3, hkv, q);
  check_scores(what, scale, logit_cap, sink, q);
  CHECK_ARG(last >= 0 && last <= INT32_MAX, what, ": last must be 0 (all new tokens) or positive, not ", last);
  CHECK_ARG(q.size(0) * q.size(1) < (int64_t(1) << 31) && batch < 65536, what, ": too many rows or requests");
  check_ints(prefix_lens, batch, "prefix_lens", q);
  check_ints(q_start, batch, "q_start_loc", q);
  c10::cuda::CUDAGuard g(q.device());
  a.index = cache_index(what, req_to_token, req_pool_indices, seq_lens, sums, q);
  a.sums = {sums.data_ptr<float>(), sums.stride(0), sums.stride(1)};
  a.prefix_lens = prefix_lens.data_ptr<int>();
  a.q_start = q_start.data_ptr<int>();
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.sink = sink.has_value() ? sink->data_ptr<float>() : nullptr;
  a.q_stride = q.stride(0);
  a.num_slots = k_cache.size(0);
  a.kv_tok_stride = k_cache.stride(0);
  a.kv_head_stride = k_cache.stride(1);
  a.rows = q.size(0);
  a.hq = static_cast<int>(q.size(1));
  a.hkv = static_cast<int>(hkv);
  a.head_dim = static_cast<int>(hd);
  a.num_sms = device_state(q.get_device()).num_sms;
  a.last = static_cast<int>(last);
  a.add = add;
  a.scale = static_cast<float>(scale);
  a.logit_cap = static_cast<float>(logit_cap);
  a.dt = dtype_of(q);
  Tensor ws = torch::empty({mb200::weights_prompt_floats(a)}, q.options().dtype(torch::kFloat32));
  a.workspace = ws.data_ptr<float>();
  const int rc = mb200::launch_weights_prompt(a, stream_of(q));
  TORCH_CHECK(rc == 0, "mllm_b200 attention_prefill_weights: unsupported configuration or launch failure (code ", rc, ")");
}

std::vector<Tensor> cache_select(const Tensor& sums, const Tensor& req_pool_indices, const Tensor& seq_lens, const Tensor& budgets, int64_t width,
                                 int64_t first, int64_t recent, int64_t pool) {
  const char* what = "cache_select";
  CHECK_ARG(sums.is_cuda() && sums.dim() == 4, what, ": sums must be a device tensor [layers, requests, heads, tokens]");
  check_sums(what, sums, 4, sums.size(2), sums);
  const int64_t batch = req_pool_indices.numel();
  check_ints(budgets, batch, "budgets", sums);
  CHECK_ARG(width >= 0 && width <= sums.size(3), what, ": max_budget must be from 0 to the ", sums.size(3), " tokens of the sums, not ", width);
  CHECK_ARG(first >= 0 && first <= INT32_MAX && recent >= 0 && recent <= INT32_MAX, what, ": first and recent are numbers of tokens");
  CHECK_ARG(pool >= 1 && pool <= 63 && pool % 2 == 1, what, ": pool must be odd and from 1 to 63, not ", pool);
  const int64_t lists = sums.size(0) * batch * sums.size(2);
  CHECK_ARG(lists < (int64_t(1) << 28), what, ": too many lists");
  c10::cuda::CUDAGuard g(sums.device());
  mb200::CacheSelectArgs a{};
  a.index = cache_index(what, c10::nullopt, req_pool_indices, seq_lens, sums, sums);
  Tensor keep = torch::empty({sums.size(0), batch, sums.size(2), width}, budgets.options()), counts = torch::empty({batch}, budgets.options());
  if (lists == 0) counts.zero_();
  a.sums = sums.data_ptr<float>();
  a.budgets = budgets.data_ptr<int>();
  a.keep = keep.data_ptr<int>();
  a.counts = counts.data_ptr<int>();
  a.layer_stride = sums.stride(0);
  a.row_stride = sums.stride(1);
  a.head_stride = sums.stride(2);
  a.layers = static_cast<int>(sums.size(0));
  a.hkv = static_cast<int>(sums.size(2));
  a.width = static_cast<int>(width);
  a.first = static_cast<int>(first);
  a.recent = static_cast<int>(recent);
  a.pool = static_cast<int>(pool);
  a.num_sms = device_state(sums.get_device()).num_sms;
  const int rc = mb200::launch_cache_select(a, stream_of(sums));
  TORCH_CHECK(rc == 0, "mllm_b200 cache_select: launch failure (code ", rc, ")");
  return {keep, counts};
}

void cache_evict(const Tensor& store, const c10::optional<Tensor>& sums, const Tensor& req_to_token, const Tensor& req_pool_indices, const Tensor& keep,
                 const Tensor& counts) {
  const char* what = "cache_evict";
  const int64_t batch = req_pool_indices.numel();
  CHECK_ARG(store.is_cuda() && store.dim() == 5 && store.size(1) == 2 && store.is_contiguous() && store.size(4) * store.element_size() % 16 == 0 &&
                (reinterpret_cast<uintptr_t>(store.data_ptr()) & 15) == 0,
            what, ": store must be a contiguous device tensor [layers, 2, heads, slots, features] with rows of 16-byte multiples");
  CHECK_ARG(keep.device() == store.device() && keep.scalar_type() == at::kInt && keep.is_contiguous() && keep.dim() == 4 && keep.size(0) == store.size(0) &&
                keep.size(1) == batch && keep.size(2) == store.size(2),
            what, ": keep must be contiguous int32 [", store.size(0), ", ", batch, ", ", store.size(2), ", tokens] on ", store.device());
  check_ints(counts, batch, "counts", store);
  const int64_t lists = keep.size(0) * batch * keep.size(2);
  CHECK_ARG(lists < (int64_t(1) << 28) && keep.size(3) < (int64_t(1) << 31) && store.size(3) < (int64_t(1) << 31) &&
                store.size(4) * store.element_size() < (int64_t(1) << 20),
            what, ": too many lists, tokens or slots, or rows too wide");
  if (sums.has_value()) {
    check_written_sums(what, *sums, 4, store.size(2), store);
    CHECK_ARG(sums->size(0) == store.size(0), what, ": sums of ", sums->size(0), " layers, and a store of ", store.size(0));
  }
  c10::cuda::CUDAGuard g(store.device());
  mb200::CacheEvictArgs a{};
  a.index = cache_index(what, req_to_token, req_pool_indices, c10::nullopt, sums, store);
  a.store = store.data_ptr();
  a.keep = keep.data_ptr<int>();
  a.counts = counts.data_ptr<int>();
  a.num_slots = store.size(3);
  if (sums.has_value()) {
    a.sums = sums->data_ptr<float>();
    a.layer_stride = sums->stride(0);
    a.row_stride = sums->stride(1);
    a.head_stride = sums->stride(2);
  }
  a.layers = static_cast<int>(store.size(0));
  a.hkv = static_cast<int>(store.size(2));
  a.width = static_cast<int>(keep.size(3));
  a.row_bytes = static_cast<int>(store.size(4) * store.element_size());
  a.num_sms = device_state(store.get_device()).num_sms;
  const int rc = mb200::launch_cache_evict(a, stream_of(store));
  TORCH_CHECK(rc == 0, "mllm_b200 cache_evict: launch failure (code ", rc, ")");
}

}  // namespace
