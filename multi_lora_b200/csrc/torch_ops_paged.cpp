// torch.ops.mlora.* of the paged serving step — a thin PyTorch binding over the
// C ABI (include/mlora_b200.h), beside torch_ops.cpp. Checks dtypes, devices,
// shapes and strides, then forwards device pointers and the current CUDA
// stream. paged_attention, verify_draft allocate only their outputs.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include "../../include/mlora_b200.h"
#include "torch_ops_paged.h"

namespace {

void on_device(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda(), "mlora: ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == dev, "mlora: ", name, " is on ", t.device(), ", expected ", dev);
}

int32_t* i32(const at::Tensor& t, const char* name, int64_t len, const at::Device& dev) {
  on_device(t, name, dev);
  TORCH_CHECK(t.scalar_type() == at::kInt, "mlora: ", name, " must be int32 (got ", t.scalar_type(), ")");
  TORCH_CHECK(t.dim() == 1 && t.is_contiguous() && t.numel() == len, "mlora: ", name, " must be a contiguous int32 [",
              len, "] (got ", t.sizes(), ")");
  return t.data_ptr<int32_t>();
}

int32_t code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MLORA_BF16;
    case at::kHalf: return MLORA_F16;
    case at::kFloat: return MLORA_F32;
    default: TORCH_CHECK(false, "mlora: unsupported dtype ", t);
  }
  return -1;
}

uint32_t* status_word(const c10::optional<at::Tensor>& status, const at::Device& dev) {
  if (!status.has_value()) return nullptr;
  on_device(*status, "status", dev);
  TORCH_CHECK(status->scalar_type() == at::kInt && status->numel() >= 1, "mlora: status must be an int32 tensor");
  return reinterpret_cast<uint32_t*>(status->data_ptr());
}

void done(int rc) { TORCH_CHECK(rc == MLORA_OK, "mlora: ", mlora_last_error()); }

// Stride of dimension d: `dense` where there is one entry, whose stride may be anything.
int64_t stride_of(const at::Tensor& t, int64_t d, int64_t dense) { return t.size(d) > 1 ? t.stride(d) : dense; }

int64_t table_rows(const at::Tensor& t, int64_t requests, const at::Device& dev) {
  on_device(t, "block_tables", dev);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == requests &&
                  (t.size(1) <= 1 || t.stride(1) == 1),
              "mlora: block_tables must be int32 [", requests, ", max_blocks] with unit column stride (got ", t.sizes(),
              ")");
  return requests > 1 ? t.stride(0) : t.size(1);
}

mlora_paged_cache_t cache_of(const at::Tensor& k, const at::Tensor& v, const at::Device& dev) {
  on_device(k, "k_cache", dev);
  on_device(v, "v_cache", dev);
  TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes(),
              "mlora: k_cache and v_cache must be [num_blocks, block_size, kv_heads, head_dim] (got ", k.sizes(), " and ",
              v.sizes(), ")");
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "mlora: k_cache and v_cache must share a dtype");
  TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, "mlora: the cache's head_dim must have unit stride");
  mlora_paged_cache_t c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.num_blocks = k.size(0);
  c.block_size = (int32_t)k.size(1);
  c.kv_heads = (int32_t)k.size(2);
  c.head_dim = (int32_t)k.size(3);
  c.dtype = code(k.scalar_type());
  c.k_block_stride = k.stride(0);
  c.k_slot_stride = k.stride(1);
  c.k_head_stride = k.stride(2);
  c.v_block_stride = v.stride(0);
  c.v_slot_stride = v.stride(1);
  c.v_head_stride = v.stride(2);
  return c;
}

}  // namespace

namespace mlora_torch {

void plan_paged_step(const at::Tensor& ctx_lens, const at::Tensor& new_lens, const at::Tensor& held_blocks,
                     const at::Tensor& free_blocks, const at::Tensor& free_head, at::Tensor block_tables,
                     int64_t block_size, at::Tensor q_indptr, at::Tensor kv_lens, at::Tensor held_out,
                     at::Tensor free_head_out, at::Tensor positions, at::Tensor slot_map, at::Tensor workspace,
                     const c10::optional<at::Tensor>& status) {
  const at::Device dev = ctx_lens.device();
  const int64_t r = ctx_lens.numel(), max_tokens = slot_map.numel();
  TORCH_CHECK(block_size >= 1 && block_size <= INT32_MAX, "mlora: block_size ", block_size, " invalid");
  const int64_t rows = table_rows(block_tables, r, dev);
  on_device(workspace, "workspace", dev);
  TORCH_CHECK(workspace.scalar_type() == at::kInt && workspace.numel() >= 1,
              "mlora: workspace must be an int32 tensor, zero before its first use");
  const c10::cuda::CUDAGuard guard(dev);
  done(mlora_plan_paged_step(
      i32(ctx_lens, "ctx_lens", r, dev), i32(new_lens, "new_lens", r, dev), i32(held_blocks, "held_blocks", r, dev), r,
      i32(free_blocks, "free_blocks", free_blocks.numel(), dev), free_blocks.numel(), i32(free_head, "free_head", 1, dev),
      block_tables.numel() > 0 ? block_tables.data_ptr<int32_t>() : nullptr, rows, block_tables.size(1),
      (int32_t)block_size, i32(q_indptr, "q_indptr", r + 1, dev), i32(kv_lens, "kv_lens", r, dev),
      i32(held_out, "plan.held_blocks", r, dev), i32(free_head_out, "plan.free_head", 1, dev),
      i32(positions, "positions", max_tokens, dev), i32(slot_map, "slot_map", max_tokens, dev), max_tokens,
      reinterpret_cast<uint32_t*>(workspace.data_ptr()), status_word(status, dev),
      at::cuda::getCurrentCUDAStream().stream()));
}

void write_paged_kv(const at::Tensor& k, const at::Tensor& v, at::Tensor k_cache, at::Tensor v_cache,
                    const at::Tensor& slot_map, const c10::optional<at::Tensor>& status) {
  const at::Device dev = k.device();
  on_device(k, "k", dev);
  on_device(v, "v", dev);
  const mlora_paged_cache_t c = cache_of(k_cache, v_cache, dev);
  TORCH_CHECK(k.dim() == 3 && k.size(1) == c.kv_heads && k.size(2) == c.head_dim && v.sizes() == k.sizes(),
              "mlora: k and v must be [tokens, ", c.kv_heads, ", ", c.head_dim, "] (got ", k.sizes(), " and ", v.sizes(),
              ")");
  TORCH_CHECK(k.scalar_type() == k_cache.scalar_type() && v.scalar_type() == k_cache.scalar_type(),
              "mlora: k, v and the cache must share a dtype");
  TORCH_CHECK(k.stride(2) == 1 && v.stride(2) == 1, "mlora: k and v must have unit stride in head_dim");
  const c10::cuda::CUDAGuard guard(dev);
  done(mlora_write_paged_kv(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), k.size(0),
                            &c, i32(slot_map, "slot_map", k.size(0), dev), status_word(status, dev),
                            at::cuda::getCurrentCUDAStream().stream()));
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_tables, const at::Tensor& kv_lens, const at::Tensor& q_indptr,
                           int64_t max_q_len, double scale, int64_t window, const c10::optional<at::Tensor>& out_,
                           const at::Tensor& workspace, const c10::optional<at::Tensor>& status) {
  const at::Device dev = q.device();
  on_device(q, "q", dev);
  const mlora_paged_cache_t c = cache_of(k_cache, v_cache, dev);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == c.head_dim && q.stride(2) == 1,
              "mlora: q must be [tokens, q_heads, ", c.head_dim, "] with unit stride in head_dim (got ", q.sizes(), ")");
  TORCH_CHECK(q.scalar_type() == k_cache.scalar_type(), "mlora: q and the cache must share a dtype");
  TORCH_CHECK(q.size(1) >= 1 && q.size(1) % c.kv_heads == 0, "mlora: ", q.size(1), " query heads over ", c.kv_heads,
              " key heads");
  const int64_t r = kv_lens.numel();
  const int64_t rows = table_rows(block_tables, r, dev);
  TORCH_CHECK(window >= 0 && window <= INT32_MAX, "mlora: window ", window, " invalid");
  on_device(workspace, "workspace", dev);
  TORCH_CHECK(workspace.is_contiguous(), "mlora: workspace must be contiguous");
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor out;
  if (out_.has_value()) {
    out = *out_;
    on_device(out, "out", dev);
    TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1,
                "mlora: out must be like q with unit stride in head_dim");
  } else {
    out = at::detail::empty_cuda(q.sizes(), q.scalar_type(), dev, c10::nullopt);
  }
  done(mlora_paged_attention(q.data_ptr(), stride_of(q, 0, c.head_dim), stride_of(q, 1, c.head_dim), q.size(0), (int32_t)q.size(1), &c,
                             block_tables.numel() > 0 ? block_tables.data_ptr<int32_t>() : nullptr, rows,
                             block_tables.size(1), i32(kv_lens, "kv_lens", r, dev),
                             i32(q_indptr, "q_indptr", r + 1, dev), r, max_q_len, (float)scale, (int32_t)window,
                             out.data_ptr(), stride_of(out, 0, c.head_dim), stride_of(out, 1, c.head_dim), workspace.data_ptr(),
                             (size_t)workspace.nbytes(), status_word(status, dev),
                             at::cuda::getCurrentCUDAStream().stream()));
  return out;
}

std::tuple<at::Tensor, at::Tensor> verify_draft(const at::Tensor& target, const c10::optional<at::Tensor>& draft,
                                                const at::Tensor& draft_tokens, const at::Tensor& row_indptr,
                                                const at::Tensor& accept_u, const at::Tensor& sample_u,
                                                const c10::optional<at::Tensor>& status) {
  const at::Device dev = target.device();
  on_device(target, "target_probs", dev);
  on_device(draft_tokens, "draft_tokens", dev);
  on_device(accept_u, "accept_u", dev);
  on_device(sample_u, "sample_u", dev);
  TORCH_CHECK(target.dim() == 2 && target.stride(1) == 1, "mlora: target_probs must be [rows, vocab] with unit column stride");
  TORCH_CHECK(draft_tokens.dim() == 2 && draft_tokens.is_contiguous() && draft_tokens.scalar_type() == at::kLong,
              "mlora: draft_tokens must be a contiguous int64 [requests, max_drafts]");
  const int64_t r = draft_tokens.size(0), k = draft_tokens.size(1), vocab = target.size(1);
  TORCH_CHECK(accept_u.scalar_type() == at::kFloat && accept_u.is_contiguous() && accept_u.sizes() == draft_tokens.sizes(),
              "mlora: accept_u must be a contiguous float32 tensor like draft_tokens");
  TORCH_CHECK(sample_u.scalar_type() == at::kFloat && sample_u.is_contiguous() && sample_u.dim() == 1 && sample_u.size(0) == r,
              "mlora: sample_u must be a contiguous float32 [", r, "]");
  if (draft.has_value()) {
    on_device(*draft, "draft_probs", dev);
    TORCH_CHECK(draft->dim() == 3 && draft->size(0) == r && draft->size(1) == k && draft->size(2) == vocab &&
                    draft->stride(2) == 1 && draft->scalar_type() == target.scalar_type(),
                "mlora: draft_probs must be [", r, ", ", k, ", ", vocab, "] of target_probs' dtype with unit stride in vocab");
  }
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor tokens = at::detail::empty_cuda({r, k + 1}, at::kLong, dev, c10::nullopt);
  at::Tensor emitted = at::detail::empty_cuda({r}, at::kInt, dev, c10::nullopt);
  done(mlora_verify_draft(target.data_ptr(), target.size(0), vocab, stride_of(target, 0, vocab),
                          draft.has_value() ? draft->data_ptr() : nullptr,
                          draft.has_value() ? stride_of(*draft, 0, k * vocab) : 0,
                          draft.has_value() ? stride_of(*draft, 1, vocab) : 0, draft_tokens.data_ptr<int64_t>(),
                          i32(row_indptr, "row_indptr", r + 1, dev), r, (int32_t)k, accept_u.data_ptr<float>(),
                          sample_u.data_ptr<float>(), tokens.data_ptr<int64_t>(), emitted.data_ptr<int32_t>(),
                          code(target.scalar_type()), status_word(status, dev),
                          at::cuda::getCurrentCUDAStream().stream()));
  return {tokens, emitted};
}

}  // namespace mlora_torch

TORCH_LIBRARY_FRAGMENT(mlora, m) {
  m.def(
      "plan_paged_step(Tensor ctx_lens, Tensor new_lens, Tensor held_blocks, Tensor free_blocks, Tensor free_head, "
      "Tensor(a!) block_tables, int block_size, Tensor(b!) q_indptr, Tensor(c!) kv_lens, Tensor(d!) held_out, "
      "Tensor(e!) free_head_out, Tensor(f!) positions, Tensor(g!) slot_map, Tensor(h!) workspace, "
      "Tensor(i!)? status=None) -> ()");
  m.def(
      "write_paged_kv(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slot_map, "
      "Tensor(c!)? status=None) -> ()");
  m.def(
      "paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor kv_lens, Tensor q_indptr, "
      "int max_q_len, float scale, int window, Tensor(a!)? out, Tensor(b!) workspace, Tensor(c!)? status=None) "
      "-> Tensor");
  m.def(
      "verify_draft(Tensor target_probs, Tensor? draft_probs, Tensor draft_tokens, Tensor row_indptr, Tensor accept_u, "
      "Tensor sample_u, Tensor(a!)? status=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mlora, CUDA, m) {
  m.impl("plan_paged_step", &mlora_torch::plan_paged_step);
  m.impl("write_paged_kv", &mlora_torch::write_paged_kv);
  m.impl("paged_attention", &mlora_torch::paged_attention);
  m.impl("verify_draft", &mlora_torch::verify_draft);
}
