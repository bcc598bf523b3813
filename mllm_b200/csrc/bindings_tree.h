// PyTorch binding of the kernels for drafted token trees, part of the module of latent attention.
#pragma once

#include <cfloat>

#include "bindings_common.h"
#include "tree.h"

// Refusals are ValueErrors, as they are for CPU tensors
#define CHECK_ARG(...) TORCH_CHECK_VALUE(__VA_ARGS__)

namespace {

void check_int_vec(const Tensor& t, int64_t n, const char* name) {
  CHECK_ARG(t.is_cuda() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == n, "mllm_b200: ", name,
              " must be a contiguous int32 device tensor of ", n, " elements");
}

void check_f32(const Tensor& t, int64_t n, const char* name, const Tensor& like) {
  CHECK_ARG(t.device() == like.device() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == n, "mllm_b200: ", name,
            " must be a contiguous fp32 vector of ", n, " elements on ", like.device());
}
void check_rows_type(const Tensor& t, const char* name) {
  CHECK_ARG(t.is_cuda() && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf), "mllm_b200: ", name,
            " must be a bf16 or fp16 device tensor");
}

mb200::TreeIndex tree_index(const Tensor& req_to_token, const Tensor& req_pool_indices, const Tensor& seq_lens, const Tensor& prefix_lens,
                            const Tensor& q_start, const Tensor& parents, int64_t rows) {
  const int64_t batch = req_pool_indices.numel();
  CHECK_ARG(rows < (int64_t(1) << 31) && batch < (int64_t(1) << 31), "mllm_b200: too many rows or requests");
  CHECK_ARG(req_to_token.is_cuda() && req_to_token.dim() == 2 && req_to_token.scalar_type() == at::kInt && req_to_token.stride(1) == 1,
              "mllm_b200: req_to_token must be a two-dimensional int32 device tensor with unit inner stride");
  check_int_vec(req_pool_indices, batch, "req_pool_indices");
  check_int_vec(seq_lens, batch, "seq_lens");
  check_int_vec(prefix_lens, batch, "prefix_lens");
  check_int_vec(q_start, batch, "q_start_loc");
  check_int_vec(parents, rows, "parents");
  for (const Tensor* t : {&req_to_token, &req_pool_indices, &seq_lens, &prefix_lens, &q_start})
    CHECK_ARG(t->device() == parents.device(), "mllm_b200: the index tensors are on different devices");
  mb200::TreeIndex ix{};
  ix.req_to_token = req_to_token.data_ptr<int>();
  ix.req_pool_indices = req_pool_indices.data_ptr<int>();
  ix.seq_lens = seq_lens.data_ptr<int>();
  ix.prefix_lens = prefix_lens.data_ptr<int>();
  ix.q_start = q_start.data_ptr<int>();
  ix.parents = parents.data_ptr<int>();
  ix.status = device_state(parents.get_device()).status.data_ptr<int>();
  ix.table_stride = req_to_token.stride(0);
  ix.table_rows = static_cast<int>(req_to_token.size(0));
  ix.table_cols = static_cast<int>(req_to_token.size(1));
  ix.rows = static_cast<int>(rows);
  ix.batch = static_cast<int>(batch);
  return ix;
}

// 0: the caches hold `dt`; 1 / 2: unscaled e4m3 / e5m2
int check_caches(const Tensor& k_cache, const Tensor& v_cache, at::ScalarType dt, int64_t hkv, int64_t head_dim, const Tensor& like) {
  const auto ct = k_cache.scalar_type();
  const int fmt = ct == dt ? 0 : ct == at::kFloat8_e4m3fn ? 1 : ct == at::kFloat8_e5m2 ? 2 : -1;
  const int64_t unit = fmt == 0 ? 8 : 16;       // elements of 16 bytes
  CHECK_ARG(fmt >= 0 && v_cache.scalar_type() == ct && k_cache.dim() == 3 && k_cache.sizes() == v_cache.sizes() &&
                  k_cache.strides() == v_cache.strides() && k_cache.stride(2) == 1 && k_cache.size(1) == hkv && k_cache.size(2) == head_dim &&
                  k_cache.stride(0) % unit == 0 && k_cache.stride(1) % unit == 0 && k_cache.device() == like.device() &&
                  v_cache.device() == like.device(),
              "kv cache: [slots, kv_heads, head_dim] views of the activation dtype, float8_e4m3fn or float8_e5m2 on the queries' device, "
              "with unit inner stride and rows on 16-byte boundaries");
  CHECK_ARG(((reinterpret_cast<uintptr_t>(k_cache.data_ptr()) | reinterpret_cast<uintptr_t>(v_cache.data_ptr())) & 15) == 0,
              "kv cache: rows must begin on 16-byte boundaries");
  return fmt;
}

Tensor attention_tree(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& req_to_token, const Tensor& req_pool_indices,
                      const Tensor& seq_lens, const Tensor& prefix_lens, const Tensor& q_start, const Tensor& parents, double scale,
                      const c10::optional<Tensor>& given, int64_t window, double logit_cap, const c10::optional<Tensor>& sink, int64_t chunk) {
  check_rows_type(q, "q");
  CHECK_ARG(q.dim() == 3 && k_cache.dim() == 3 && q.stride(2) == 1 && q.stride(1) == q.size(2) && q.stride(0) % 8 == 0,
            "attention_tree: q must be [T,Hq,D], heads of a node contiguous, rows on 16-byte boundaries");
  const int64_t hd = q.size(2);
  CHECK_ARG(hd == 64 || hd == 128 || hd == 256, "attention_tree: heads of 64, 128 or 256 features, not ", hd);
  CHECK_ARG(window >= 0 && chunk >= 0 && (window == 0 || chunk == 0) && window < (1 << 30) && chunk < (1 << 30),
            "attention_tree: either a sliding window or chunks, of positive lengths");
  // a row's maximum is taken before its scores are scaled, and a score of minus infinity has to stay one
  CHECK_ARG(scale >= FLT_MIN && scale <= FLT_MAX, "attention_tree: scale must be positive and finite, not ", scale);
  Tensor out = given.has_value() ? *given : torch::empty(q.sizes(), q.options());
  CHECK_ARG(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device() && out.stride(2) == 1 &&
                out.stride(1) == hd && out.stride(0) % 8 == 0,
            "attention_tree: out must be [T,Hq,D] like q, heads of a node contiguous, rows on 16-byte boundaries");
  CHECK_ARG(((reinterpret_cast<uintptr_t>(q.data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) & 15) == 0,
            "attention_tree: q and out must begin on 16-byte boundaries");
  c10::cuda::CUDAGuard g(q.device());
  CHECK_ARG(parents.device() == q.device(), "attention_tree: q and parents are on different devices");
  mb200::TreeAttnArgs a{};
  a.index = tree_index(req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start, parents, q.size(0));
  a.hq = static_cast<int>(q.size(1));
  a.hkv = static_cast<int>(k_cache.size(1));
  a.head_dim = static_cast<int>(hd);
  a.kv_fmt = check_caches(k_cache, v_cache, q.scalar_type(), a.hkv, hd, q);
  CHECK_ARG(a.hkv > 0 && a.hq > 0 && a.hq % a.hkv == 0 && a.hq / a.hkv <= 128, "attention_tree: ", a.hq, " query heads over ", a.hkv, " kv heads");
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.out = out.data_ptr();
  if (sink.has_value()) {
    check_f32(*sink, a.hq, "sink", q);
    a.sink = sink->data_ptr<float>();
  }
  a.q_stride = q.stride(0);
  a.out_stride = out.stride(0);
  a.num_slots = k_cache.size(0);
  a.kv_tok_stride = k_cache.stride(0);
  a.kv_head_stride = k_cache.stride(1);
  a.window = static_cast<int>(window);
  a.chunk = static_cast<int>(chunk);
  a.scale = static_cast<float>(scale);
  a.logit_cap = static_cast<float>(logit_cap);
  a.dt = dtype_of(q);
  a.plan = mb200::tree_plan(a.head_dim, a.hq / a.hkv, q.size(0), a.index.batch, device_state(q.get_device()).num_sms);
  // of this call alone: the caching allocator hands it out again in stream order, and a captured graph has its own
  Tensor ws = torch::empty({a.plan.workspace_floats}, q.options().dtype(torch::kFloat32));
  a.workspace = ws.data_ptr<float>();
  const int rc = mb200::launch_attention_tree(a, stream_of(q));
  TORCH_CHECK(rc == 0, "mllm_b200 attention_tree: unsupported configuration or launch failure (code ", rc, ")");
  return out;
}

void check_gain(const c10::optional<Tensor>& g, const Tensor& like, int64_t n, const char* name) {
  if (!g.has_value()) return;
  CHECK_ARG(g->device() == like.device() && g->scalar_type() == like.scalar_type() && g->is_contiguous() && g->numel() == n, "mllm_b200: ",
              name, " must be a contiguous vector of ", n, " elements like the rows");
  CHECK_ARG((reinterpret_cast<uintptr_t>(g->data_ptr()) & 15) == 0, "mllm_b200: ", name, " must begin on a 16-byte boundary");
}

Tensor tree_qk_norm_rope_kv_write(const Tensor& qkv, const c10::optional<Tensor>& q_gain, const c10::optional<Tensor>& k_gain,
                                  const Tensor& parents, const Tensor& req_to_token, const Tensor& req_pool_indices, const Tensor& seq_lens,
                                  const Tensor& prefix_lens, const Tensor& q_start, const Tensor& inv_freq, Tensor& k_cache, Tensor& v_cache,
                                  int64_t hq, int64_t hkv, int64_t hd, double eps, const c10::optional<Tensor>& delta) {
  check_rows_type(qkv, "qkv");
  CHECK_ARG(hq > 0 && hkv > 0, "tree_qk_norm_rope_kv_write: ", hq, " query heads and ", hkv, " key heads");
  CHECK_ARG((hd == 64 || hd == 128 || hd == 256) && qkv.dim() == 2 && qkv.stride(1) == 1 && qkv.size(1) == (hq + 2 * hkv) * hd &&
                  qkv.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(qkv.data_ptr()) & 15) == 0,
              "qkv must be [T, (Hq + 2 Hkv) * D], D 64, 128 or 256, rows on 16-byte boundaries");
  CHECK_ARG(parents.device() == qkv.device() && inv_freq.device() == qkv.device(), "mllm_b200: tensors on different devices");
  CHECK_ARG(inv_freq.scalar_type() == at::kFloat && inv_freq.is_contiguous() && inv_freq.numel() * 2 <= hd && inv_freq.numel() % 8 == 0,
              "inv_freq must be fp32, one per rotated pair, a multiple of 8");
  check_gain(q_gain, qkv, hd, "q_weight");
  check_gain(k_gain, qkv, hd, "k_weight");
  c10::cuda::CUDAGuard g(qkv.device());
  mb200::TreePrologueArgs a{};
  a.index = tree_index(req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start, parents, qkv.size(0));
  a.kv_fmt = check_caches(k_cache, v_cache, qkv.scalar_type(), hkv, hd, qkv);
  if (delta.has_value()) {
    check_int_vec(*delta, req_pool_indices.numel(), "position_delta");
    CHECK_ARG(delta->device() == qkv.device(), "mllm_b200: tensors on different devices");
    a.position_delta = delta->data_ptr<int>();
  }
  Tensor q = torch::empty({qkv.size(0), hq, hd}, qkv.options());
  a.qkv = qkv.data_ptr();
  a.q_gain = q_gain.has_value() ? q_gain->data_ptr() : nullptr;
  a.k_gain = k_gain.has_value() ? k_gain->data_ptr() : nullptr;
  a.inv_freq = inv_freq.data_ptr<float>();
  a.q_out = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.qkv_stride = qkv.stride(0);
  a.kv_tok_stride = k_cache.stride(0);
  a.kv_head_stride = k_cache.stride(1);
  a.num_slots = k_cache.size(0);
  a.hq = static_cast<int>(hq);
  a.hkv = static_cast<int>(hkv);
  a.head_dim = static_cast<int>(hd);
  a.rotated = static_cast<int>(inv_freq.numel() * 2);
  a.eps = static_cast<float>(eps);
  a.dt = dtype_of(qkv);
  const int rc = mb200::launch_tree_prologue(a, stream_of(qkv));
  TORCH_CHECK(rc == 0, "mllm_b200 tree_qk_norm_rope_kv_write: launch failure (code ", rc, ")");
  return q;
}

void tree_kv_compact(Tensor& store, const Tensor& req_to_token, const Tensor& req_pool_indices, const Tensor& prefix_lens, const Tensor& path,
                     const Tensor& counts) {
  const int64_t batch = req_pool_indices.numel(), row = store.size(-1) * store.element_size();
  CHECK_ARG(store.is_cuda() && store.dim() >= 2 && store.is_contiguous() && row % 16 == 0 &&
                  (reinterpret_cast<uintptr_t>(store.data_ptr()) & 15) == 0,
              "tree_kv_compact: store must be contiguous [.., slots, features] with rows of 16-byte multiples");
  CHECK_ARG(req_to_token.is_cuda() && req_to_token.dim() == 2 && req_to_token.scalar_type() == at::kInt && req_to_token.stride(1) == 1,
              "mllm_b200: req_to_token must be a two-dimensional int32 device tensor with unit inner stride");
  CHECK_ARG(path.dim() == 2 && path.size(0) == batch, "mllm_b200: path must be [requests, steps]");
  check_int_vec(req_pool_indices, batch, "req_pool_indices");
  check_int_vec(prefix_lens, batch, "prefix_lens");
  check_int_vec(path, batch * path.size(1), "path");
  check_int_vec(counts, batch, "counts");
  for (const Tensor* t : {&req_to_token, &req_pool_indices, &prefix_lens, &path, &counts})
    CHECK_ARG(t->device() == store.device(), "mllm_b200: tensors on different devices");
  if (store.numel() == 0 || batch == 0) return;
  const int64_t planes = store.numel() / (store.size(-2) * store.size(-1));
  CHECK_ARG(planes * (row / 16) < (int64_t(1) << 31) - (int64_t(1) << 24), "tree_kv_compact: ", planes, " planes of rows of ", row, " bytes are too many");
  c10::cuda::CUDAGuard g(store.device());
  mb200::TreeCompactArgs a{};
  a.store = store.data_ptr();
  a.req_to_token = req_to_token.data_ptr<int>();
  a.req_pool_indices = req_pool_indices.data_ptr<int>();
  a.prefix_lens = prefix_lens.data_ptr<int>();
  a.path = path.data_ptr<int>();
  a.counts = counts.data_ptr<int>();
  a.status = device_state(store.get_device()).status.data_ptr<int>();
  a.table_stride = req_to_token.stride(0);
  a.num_slots = store.size(-2);
  a.batch = static_cast<int>(batch);
  a.steps = static_cast<int>(path.size(1));
  a.table_rows = static_cast<int>(req_to_token.size(0));
  a.table_cols = static_cast<int>(req_to_token.size(1));
  a.planes = static_cast<int>(planes);
  a.row_bytes = static_cast<int>(row);
  const int rc = mb200::launch_tree_compact(a, stream_of(store));
  TORCH_CHECK(rc == 0, "mllm_b200 tree_kv_compact: unsupported configuration or launch failure (code ", rc, ")");
}

std::vector<Tensor> tree_speculative_sample(const Tensor& logits, const Tensor& tokens, const Tensor& parents, const Tensor& tree_lens,
                                            const Tensor& q_start, const Tensor& temperature, const Tensor& top_k, const Tensor& top_p,
                                            const c10::optional<Tensor>& min_p, const Tensor& uniform, const Tensor& uniform_final,
                                            int64_t steps, const c10::optional<Tensor>& draft) {
  CHECK_ARG(logits.is_cuda() && (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf || logits.scalar_type() == at::kFloat),
            "logits must be a bf16, fp16 or fp32 device tensor");
  CHECK_ARG(logits.dim() == 2 && logits.stride(1) == 1, "logits must be [T, vocab] with unit inner stride");
  const int64_t rows = logits.size(0), vocab = logits.size(1), batch = tree_lens.numel();
  CHECK_ARG(tokens.is_cuda() && tokens.scalar_type() == at::kLong && tokens.is_contiguous() && tokens.numel() == rows,
              "tokens must be a contiguous int64 device vector, one per row");
  check_int_vec(parents, rows, "parents");
  check_int_vec(tree_lens, batch, "tree_lens");
  check_int_vec(q_start, batch, "q_start_loc");
  check_int_vec(top_k, batch, "top_k");
  check_f32(temperature, batch, "temperature", logits);
  check_f32(top_p, batch, "top_p", logits);
  check_f32(uniform, rows, "uniform", logits);
  check_f32(uniform_final, batch, "uniform_final", logits);
  for (const Tensor* t : {&tokens, &parents, &tree_lens, &q_start, &top_k})
    CHECK_ARG(t->device() == logits.device(), "mllm_b200: tensors on different devices");
  mb200::TreeSampleArgs a{};
  if (min_p.has_value()) {
    check_f32(*min_p, batch, "min_p", logits);
    a.min_p = min_p->data_ptr<float>();
  }
  if (draft.has_value()) {
    CHECK_ARG(draft->device() == logits.device() && draft->scalar_type() == at::kFloat && draft->dim() == 2 && draft->stride(1) == 1 &&
                    draft->size(0) == rows && draft->size(1) == vocab,
                "draft_probs must be fp32 [T, vocab] with unit inner stride");
    a.draft = draft->data_ptr<float>();
    a.draft_stride = draft->stride(0);
  }
  a.dt = dtype_of(logits);
  CHECK_ARG(steps > 0 && steps < (int64_t(1) << 30), "max_steps must be positive");
  CHECK_ARG(vocab > 0 && vocab <= mb200::tree_sample_max_vocab(a.dt), "tree_speculative_sample: vocabularies of 1 to ",
              mb200::tree_sample_max_vocab(a.dt), " tokens, not ", vocab);
  c10::cuda::CUDAGuard g(logits.device());
  Tensor path = torch::empty({batch, steps}, parents.options()), out = torch::empty({batch, steps}, tokens.options()),
         counts = torch::empty({batch}, parents.options());
  a.logits = logits.data_ptr();
  a.tokens = tokens.data_ptr<int64_t>();
  a.parents = parents.data_ptr<int>();
  a.tree_lens = tree_lens.data_ptr<int>();
  a.q_start = q_start.data_ptr<int>();
  a.temperature = temperature.data_ptr<float>();
  a.top_k = top_k.data_ptr<int>();
  a.top_p = top_p.data_ptr<float>();
  a.uniform = uniform.data_ptr<float>();
  a.uniform_final = uniform_final.data_ptr<float>();
  a.path = path.data_ptr<int>();
  a.out = out.data_ptr<int64_t>();
  a.counts = counts.data_ptr<int>();
  a.status = device_state(logits.get_device()).status.data_ptr<int>();
  a.logit_stride = logits.stride(0);
  a.rows = static_cast<int>(rows);
  a.batch = static_cast<int>(batch);
  a.vocab = static_cast<int>(vocab);
  a.steps = static_cast<int>(steps);
  a.num_sms = device_state(logits.get_device()).num_sms;
  const int rc = mb200::launch_tree_sample(a, stream_of(logits));
  TORCH_CHECK(rc == 0, "mllm_b200 tree_speculative_sample: unsupported configuration or launch failure (code ", rc, ")");
  return {path, out, counts};
}

}  // namespace
