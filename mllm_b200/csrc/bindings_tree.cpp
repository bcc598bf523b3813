// PyTorch binding of the kernels for drafted token trees.
#include "bindings_common.h"
#include "tree.h"

namespace {

void check_int_vec(const Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == n, "mllm_b200: ", name,
              " must be a contiguous int32 device tensor of ", n, " elements");
}

mb200::TreeIndex tree_index(const Tensor& req_to_token, const Tensor& req_pool_indices, const Tensor& seq_lens, const Tensor& prefix_lens,
                            const Tensor& q_start, const Tensor& parents, int64_t rows) {
  const int64_t batch = req_pool_indices.numel();
  TORCH_CHECK(req_to_token.is_cuda() && req_to_token.dim() == 2 && req_to_token.scalar_type() == at::kInt && req_to_token.stride(1) == 1,
              "mllm_b200: req_to_token must be a two-dimensional int32 device tensor with unit inner stride");
  check_int_vec(req_pool_indices, batch, "req_pool_indices");
  check_int_vec(seq_lens, batch, "seq_lens");
  check_int_vec(prefix_lens, batch, "prefix_lens");
  check_int_vec(q_start, batch, "q_start_loc");
  check_int_vec(parents, rows, "parents");
  for (const Tensor* t : {&req_to_token, &req_pool_indices, &seq_lens, &prefix_lens, &q_start})
    TORCH_CHECK(t->device() == parents.device(), "mllm_b200: the index tensors are on different devices");
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
  TORCH_CHECK(fmt >= 0 && v_cache.scalar_type() == ct && k_cache.dim() == 3 && k_cache.sizes() == v_cache.sizes() &&
                  k_cache.strides() == v_cache.strides() && k_cache.stride(2) == 1 && k_cache.size(1) == hkv && k_cache.size(2) == head_dim &&
                  k_cache.stride(0) % unit == 0 && k_cache.stride(1) % unit == 0 && k_cache.device() == like.device() &&
                  v_cache.device() == like.device(),
              "kv cache: [slots, kv_heads, head_dim] views of the activation dtype, float8_e4m3fn or float8_e5m2 on the queries' device, "
              "with unit inner stride and rows on 16-byte boundaries");
  TORCH_CHECK(((reinterpret_cast<uintptr_t>(k_cache.data_ptr()) | reinterpret_cast<uintptr_t>(v_cache.data_ptr())) & 15) == 0,
              "kv cache: rows must begin on 16-byte boundaries");
  return fmt;
}

void attention_tree(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& req_to_token, const Tensor& req_pool_indices,
                    const Tensor& seq_lens, const Tensor& prefix_lens, const Tensor& q_start, const Tensor& parents, double scale, Tensor& out,
                    int64_t window, double logit_cap, const c10::optional<Tensor>& sink, int64_t chunk) {
  check_half(q, "q");
  const int64_t hd = q.size(2);
  TORCH_CHECK(q.dim() == 3 && (hd == 64 || hd == 128 || hd == 256) && q.stride(2) == 1 && q.stride(1) == hd && q.stride(0) % 8 == 0,
              "q must be [T,Hq,D], heads of a node contiguous, D 64, 128 or 256");
  TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device() && out.stride(2) == 1 &&
                  out.stride(1) == hd && out.stride(0) % 8 == 0,
              "out must be [T,Hq,D] like q, heads of a node contiguous");
  TORCH_CHECK(((reinterpret_cast<uintptr_t>(q.data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) & 15) == 0,
              "q and out must begin on 16-byte boundaries");
  c10::cuda::CUDAGuard g(q.device());
  TORCH_CHECK(parents.device() == q.device(), "attention_tree: q and parents are on different devices");
  mb200::TreeAttnArgs a{};
  a.index = tree_index(req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start, parents, q.size(0));
  a.hq = static_cast<int>(q.size(1));
  a.hkv = static_cast<int>(k_cache.size(1));
  a.head_dim = static_cast<int>(hd);
  a.kv_fmt = check_caches(k_cache, v_cache, q.scalar_type(), a.hkv, hd, q);
  TORCH_CHECK(a.hkv > 0 && a.hq % a.hkv == 0 && a.hq / a.hkv <= 128, "attention_tree: ", a.hq, " query heads over ", a.hkv, " kv heads");
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.out = out.data_ptr();
  if (sink.has_value()) {
    check_f32_vec(*sink, a.hq, "sink");
    TORCH_CHECK(sink->device() == q.device(), "attention_tree: q and sink are on different devices");
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
  a.ctas = mb200::tree_ctas(a.head_dim, device_state(q.get_device()).num_sms);
  // of this call alone: the caching allocator hands it out again in stream order, and a captured graph has its own
  Tensor ws = torch::empty({mb200::tree_workspace_floats(a.head_dim, a.hq / a.hkv, q.size(0), a.ctas)}, q.options().dtype(torch::kFloat32));
  a.workspace = ws.data_ptr<float>();
  const int rc = mb200::launch_attention_tree(a, stream_of(q));
  TORCH_CHECK(rc == 0, "mllm_b200 attention_tree: unsupported configuration or launch failure (code ", rc, ")");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("attention_tree", &attention_tree);
  m.def("read_status", &read_status);
  m.def("launch_count", &launch_count);
}
