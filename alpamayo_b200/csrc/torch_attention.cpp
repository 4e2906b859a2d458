// torch_attention.cpp — torch operators of the attention and int8 key/value
// cache entry points (include/paro_b200.h), in the same manner as
// torch_ops.cpp: outputs and workspaces from the caching allocator, launched
// on the current stream, no synchronisation, RuntimeError on bad arguments.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/paro_b200.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

paro_stream_t cur_stream() { return reinterpret_cast<paro_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }

void check_status(int s, const char* what) {
  TORCH_CHECK(s == PARO_OK, "paro_b200::", what, " failed: ", paro_status_string(s),
              (s == PARO_ERR_CUDA ? std::string(" (") + paro_last_cuda_error() + ")" : std::string()));
}

int dtype_of(at::ScalarType t, bool with_f32) {
  if (t == at::kHalf) return PARO_F16;
  if (t == at::kBFloat16) return PARO_BF16;
  TORCH_CHECK(with_f32 && t == at::kFloat, "paro_b200: unsupported dtype ", t,
              with_f32 ? " (Float, Half, BFloat16)" : " (Half, BFloat16)");
  return PARO_F32;
}

// A tensor that is read through strides: on the device, last dimension contiguous.
void check_view(const at::Tensor& t, const char* name, int64_t dims, const at::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "paro_b200: ", name, " must be a CUDA tensor on the same device");
  TORCH_CHECK(t.dim() == dims, "paro_b200: ", name, " must have ", dims, " dimensions");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), "paro_b200: ", name, " has another dtype");
  TORCH_CHECK(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, "paro_b200: ", name,
              " must be contiguous along its last dimension");
}

void check_whole(const at::Tensor& t, const char* name, at::ScalarType type, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, "paro_b200: ", name, " must be a CUDA tensor on the same device");
  TORCH_CHECK(t.scalar_type() == type, "paro_b200: ", name, " must be ", type);
  TORCH_CHECK(t.is_contiguous(), "paro_b200: ", name, " must be contiguous");
}

// Stride of a dimension; one of a single element is never used, so any
// value that the entry points accept does.
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) <= 1 ? 0 : t.stride(d); }

struct Cache {
  paro_kv8_cache c;
  const int32_t* table;
  int width;
  int64_t B;
};

Cache cache_of(const at::Tensor& k_codes, const at::Tensor& v_codes, const at::Tensor& k_scale,
               const at::Tensor& v_scale, const at::Tensor& table) {
  const at::Device dev = k_codes.device();
  check_whole(k_codes, "k_codes", at::kChar, dev);
  check_whole(v_codes, "v_codes", at::kChar, dev);
  check_whole(k_scale, "k_scale", at::kFloat, dev);
  check_whole(v_scale, "v_scale", at::kFloat, dev);
  check_whole(table, "page_table", at::kInt, dev);
  TORCH_CHECK(k_codes.dim() == 4 && v_codes.sizes() == k_codes.sizes(),
              "paro_b200: k_codes and v_codes must be int8 [pages, kv_heads, page_size, head_dim]");
  TORCH_CHECK(k_scale.dim() == 2 && k_scale.size(0) == k_codes.size(0) && k_scale.size(1) == k_codes.size(1) &&
                  v_scale.sizes() == k_scale.sizes(),
              "paro_b200: k_scale and v_scale must be float32 [pages, kv_heads]");
  TORCH_CHECK(table.dim() == 2 && table.size(1) > 0, "paro_b200: page_table must be int32 [B, pages per sequence]");
  TORCH_CHECK(k_codes.size(1) <= INT32_MAX && k_codes.size(2) <= INT32_MAX && k_codes.size(3) <= INT32_MAX &&
                  table.size(0) <= INT32_MAX && table.size(1) <= INT32_MAX,
              "paro_b200: cache too large");
  Cache r;
  r.c = paro_kv8_cache{k_codes.data_ptr<int8_t>(), v_codes.data_ptr<int8_t>(), k_scale.data_ptr<float>(),
                       v_scale.data_ptr<float>(), k_codes.size(0), (int)k_codes.size(1), (int)k_codes.size(2),
                       (int)k_codes.size(3)};
  r.table = table.data_ptr<int32_t>();
  r.width = (int)table.size(1);
  r.B = table.size(0);
  return r;
}

void check_lens(const at::Tensor& t, const char* name, int64_t n, const at::Device& dev) {
  check_whole(t, name, at::kInt, dev);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n, "paro_b200: ", name, " must be int32 [", n, "]");
}

at::Tensor attention_prefill(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu,
                             const OptTensor& cu_k_opt, double scale) {
  check_view(q, "q", 3, q);
  check_view(k, "k", 3, q);
  check_view(v, "v", 3, q);
  const int dt = dtype_of(q.scalar_type(), false);
  const at::Tensor& cu_k = cu_k_opt.has_value() && cu_k_opt->defined() ? *cu_k_opt : cu;
  TORCH_CHECK(cu.dim() == 1 && cu.size(0) >= 1 && cu.size(0) <= INT32_MAX, "paro_b200: cu_seqlens must be int32 [B + 1]");
  check_lens(cu, "cu_seqlens", cu.size(0), q.device());
  check_lens(cu_k, "cu_seqlens_k", cu.size(0), q.device());
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(2) == q.size(2), "paro_b200: k and v must be [k_rows, kv_heads, head_dim]");
  TORCH_CHECK(&cu_k != &cu || k.size(0) == q.size(0), "paro_b200: q and k have different rows and no cu_seqlens_k");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  const int64_t strides[6] = {stride_of(q, 0), stride_of(q, 1), stride_of(k, 0), stride_of(k, 1), stride_of(v, 0),
                              stride_of(v, 1)};
  const int B = (int)cu.size(0) - 1;
  const size_t wsb = paro_attention_prefill_workspace_size(B, q.size(0), k.size(0), (int)q.size(1), (int)q.size(2));
  at::Tensor ws;   // allocations start on 512-byte boundaries
  if (wsb) ws = at::empty({(int64_t)wsb}, q.options().dtype(at::kByte));
  check_status(paro_attention_prefill_ws(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, strides, cu.data_ptr<int32_t>(),
                                         cu_k.data_ptr<int32_t>(), B, q.size(0), k.size(0), (int)q.size(1),
                                         (int)k.size(1), (int)q.size(2), (float)scale, out.data_ptr(),
                                         wsb ? ws.data_ptr() : nullptr, wsb, cur_stream()),
               "attention_prefill");
  return out;
}

void kv8_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, const at::Tensor& starts,
                const at::Tensor& k_codes, const at::Tensor& v_codes, const at::Tensor& k_scale,
                const at::Tensor& v_scale, const at::Tensor& table) {
  check_view(k, "k", 3, k);
  check_view(v, "v", 3, k);
  const int dt = dtype_of(k.scalar_type(), true);
  Cache c = cache_of(k_codes, v_codes, k_scale, v_scale, table);
  TORCH_CHECK(k.device() == k_codes.device(), "paro_b200: k must be on the cache's device");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(1) == c.c.kv_heads && k.size(2) == c.c.head_dim,
              "paro_b200: k and v must be [rows, kv_heads, head_dim] of the cache");
  check_lens(cu, "cu_seqlens", c.B + 1, k.device());
  check_lens(starts, "starts", c.B, k.device());
  c10::cuda::CUDAGuard guard(k.device());
  const int64_t strides[4] = {stride_of(k, 0), stride_of(k, 1), stride_of(v, 0), stride_of(v, 1)};
  check_status(paro_kv8_append(&c.c, c.table, c.width, k.data_ptr(), v.data_ptr(), dt, strides, cu.data_ptr<int32_t>(),
                               starts.data_ptr<int32_t>(), (int)c.B, k.size(0), cur_stream()),
               "kv8_append");
}

std::tuple<at::Tensor, at::Tensor> kv8_gather(const at::Tensor& k_codes, const at::Tensor& v_codes,
                                              const at::Tensor& k_scale, const at::Tensor& v_scale,
                                              const at::Tensor& table, const at::Tensor& starts, const at::Tensor& cu,
                                              int64_t rows, at::ScalarType dtype) {
  Cache c = cache_of(k_codes, v_codes, k_scale, v_scale, table);
  check_lens(cu, "cu_seqlens", c.B + 1, k_codes.device());
  check_lens(starts, "starts", c.B, k_codes.device());
  const int dt = dtype_of(dtype, true);
  TORCH_CHECK(rows >= 0, "paro_b200: rows must not be negative");
  c10::cuda::CUDAGuard guard(k_codes.device());
  at::Tensor k = at::empty({rows, c.c.kv_heads, c.c.head_dim}, k_codes.options().dtype(dtype));
  at::Tensor v = at::empty_like(k);
  check_status(paro_kv8_gather(&c.c, c.table, c.width, starts.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), (int)c.B,
                               rows, k.data_ptr(), v.data_ptr(), dt, cur_stream()),
               "kv8_gather");
  return {k, v};
}

at::Tensor attention_kv8(const at::Tensor& q, const at::Tensor& k_codes, const at::Tensor& v_codes,
                         const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& table,
                         const at::Tensor& lens, double scale, const OptTensor& weights, const OptTensor& weights_out) {
  check_view(q, "q", 4, q);
  const int dt = dtype_of(q.scalar_type(), false);
  Cache c = cache_of(k_codes, v_codes, k_scale, v_scale, table);
  TORCH_CHECK(q.device() == k_codes.device(), "paro_b200: q must be on the cache's device");
  TORCH_CHECK(q.size(0) == c.B && q.size(3) == c.c.head_dim, "paro_b200: q must be [B, T, heads, head_dim] of the cache");
  TORCH_CHECK(q.size(1) <= INT32_MAX && q.size(2) <= INT32_MAX, "paro_b200: q too large");
  check_lens(lens, "seq_lens", c.B, q.device());
  const bool with = weights.has_value() && weights->defined();
  TORCH_CHECK(with == (weights_out.has_value() && weights_out->defined()),
              "paro_b200: weights and weights_out go together");
  const float* wi = nullptr;
  float* wo = nullptr;
  int64_t cap = 0;
  if (with) {
    check_whole(*weights, "weights", at::kFloat, q.device());
    check_whole(*weights_out, "weights_out", at::kFloat, q.device());
    TORCH_CHECK(weights->dim() == 3 && weights->size(0) == c.B && weights->size(1) == c.c.kv_heads &&
                    weights_out->sizes() == weights->sizes(),
                "paro_b200: weights must be float32 [B, kv_heads, capacity]");
    cap = weights->size(2);
    wi = weights->data_ptr<float>();
    wo = weights_out->data_ptr<float>();
  }
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (out.numel() == 0) return out;
  const int64_t strides[3] = {stride_of(q, 0), stride_of(q, 1), stride_of(q, 2)};
  const size_t wsb = paro_attention_kv8_workspace_size(&c.c, c.width, (int)c.B, (int)q.size(1), (int)q.size(2), with);
  // allocations start on 512-byte boundaries, so the workspace is aligned
  at::Tensor ws = at::empty({(int64_t)wsb}, q.options().dtype(at::kByte));
  check_status(paro_attention_kv8(&c.c, c.table, c.width, q.data_ptr(), dt, strides, (int)c.B, (int)q.size(1),
                                  (int)q.size(2), lens.data_ptr<int32_t>(), (float)scale, wi, wo, cap, out.data_ptr(),
                                  wsb ? ws.data_ptr() : out.data_ptr(), wsb, cur_stream()),
               "attention_kv8");
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> kv8_evict(const at::Tensor& weights, const at::Tensor& k_codes,
                                                         const at::Tensor& v_codes, const at::Tensor& k_scale,
                                                         const at::Tensor& v_scale, const at::Tensor& table,
                                                         const at::Tensor& lens, const at::Tensor& out_table,
                                                         int64_t budget, int64_t sink, int64_t recent) {
  Cache c = cache_of(k_codes, v_codes, k_scale, v_scale, table);
  check_whole(weights, "weights", at::kFloat, k_codes.device());
  check_whole(out_table, "out_table", at::kInt, k_codes.device());
  check_lens(lens, "seq_lens", c.B, k_codes.device());
  TORCH_CHECK(weights.dim() == 3 && weights.size(0) == c.B && weights.size(1) == c.c.kv_heads,
              "paro_b200: weights must be float32 [B, kv_heads, capacity]");
  TORCH_CHECK(out_table.dim() == 2 && out_table.size(0) == c.B && out_table.size(1) <= INT32_MAX,
              "paro_b200: out_table must be int32 [B, pages per sequence]");
  TORCH_CHECK(budget > 0 && budget <= INT32_MAX && sink >= 0 && recent >= 0 && sink <= budget && recent <= budget - sink,
              "paro_b200: budget must be positive and hold sink + recent tokens");
  c10::cuda::CUDAGuard guard(k_codes.device());
  at::Tensor kept = at::empty({c.B, c.c.kv_heads, budget}, lens.options());
  at::Tensor nw = at::empty({c.B, c.c.kv_heads, budget}, weights.options());
  at::Tensor nl = at::empty({c.B}, lens.options());
  check_status(paro_kv8_evict(&c.c, c.table, c.width, weights.data_ptr<float>(), weights.size(2),
                              lens.data_ptr<int32_t>(), (int)c.B, (int)budget, (int)sink, (int)recent,
                              kept.data_ptr<int32_t>(), nw.data_ptr<float>(), nl.data_ptr<int32_t>(),
                              out_table.data_ptr<int32_t>(), (int)out_table.size(1), cur_stream()),
               "kv8_evict");
  return {kept, nw, nl};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(paro_b200, m) {
  m.def("attention_prefill(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens, Tensor? cu_seqlens_k, float scale) -> Tensor");
  m.def("kv8_append(Tensor k, Tensor v, Tensor cu_seqlens, Tensor starts, Tensor(a!) k_codes, Tensor(b!) v_codes, "
        "Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor page_table) -> ()");
  m.def("kv8_gather(Tensor k_codes, Tensor v_codes, Tensor k_scale, Tensor v_scale, Tensor page_table, Tensor starts, "
        "Tensor cu_seqlens, int rows, ScalarType dtype) -> (Tensor, Tensor)");
  m.def("attention_kv8(Tensor q, Tensor k_codes, Tensor v_codes, Tensor k_scale, Tensor v_scale, Tensor page_table, "
        "Tensor seq_lens, float scale, Tensor? weights, Tensor(a!)? weights_out) -> Tensor");
  m.def("kv8_evict(Tensor weights, Tensor(a!) k_codes, Tensor(b!) v_codes, Tensor(c!) k_scale, Tensor(d!) v_scale, "
        "Tensor page_table, Tensor seq_lens, Tensor out_table, int budget, int sink, int recent) -> "
        "(Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(paro_b200, CUDA, m) {
  m.impl("attention_prefill", &attention_prefill);
  m.impl("kv8_append", &kv8_append);
  m.impl("kv8_gather", &kv8_gather);
  m.impl("attention_kv8", &attention_kv8);
  m.impl("kv8_evict", &kv8_evict);
}
