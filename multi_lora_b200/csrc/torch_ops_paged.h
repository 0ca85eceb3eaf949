// The operators of the paged serving step as C++ functions, what torch.ops.mlora.* of the same names run.
#pragma once

#include <ATen/ATen.h>

#include <tuple>

namespace mlora_torch {

void plan_paged_step(const at::Tensor& ctx_lens, const at::Tensor& new_lens, const at::Tensor& held_blocks,
                     const at::Tensor& free_blocks, const at::Tensor& free_head, at::Tensor block_tables,
                     int64_t block_size, at::Tensor q_indptr, at::Tensor kv_lens, at::Tensor held_out,
                     at::Tensor free_head_out, at::Tensor positions, at::Tensor slot_map, at::Tensor workspace,
                     const c10::optional<at::Tensor>& status);

void write_paged_kv(const at::Tensor& k, const at::Tensor& v, at::Tensor k_cache, at::Tensor v_cache,
                    const at::Tensor& slot_map, const c10::optional<at::Tensor>& status);

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_tables, const at::Tensor& kv_lens, const at::Tensor& q_indptr,
                           int64_t max_q_len, double scale, int64_t window, const c10::optional<at::Tensor>& out,
                           const at::Tensor& workspace, const c10::optional<at::Tensor>& status);

// The same over a cache of e4m3 codes with float32 scales [num_blocks, kv_heads].
at::Tensor paged_attention_8bit(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& block_tables,
                                const at::Tensor& kv_lens, const at::Tensor& q_indptr, int64_t max_q_len, double scale,
                                int64_t window, const c10::optional<at::Tensor>& out, const at::Tensor& workspace,
                                const c10::optional<at::Tensor>& status);

at::Tensor rotate(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& turns, bool interleaved,
                  double factor, const c10::optional<at::Tensor>& out);

// Returns the rotated queries, an undefined tensor without queries.
at::Tensor append_paged_kv(const at::Tensor& k, const at::Tensor& v, at::Tensor k_cache, at::Tensor v_cache,
                           const at::Tensor& slot_map, const c10::optional<at::Tensor>& positions,
                           const c10::optional<at::Tensor>& turns, bool interleaved, double factor,
                           const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& q_out,
                           const c10::optional<at::Tensor>& k_scales, const c10::optional<at::Tensor>& v_scales,
                           const c10::optional<at::Tensor>& status);

std::tuple<at::Tensor, at::Tensor> verify_draft(const at::Tensor& target, const c10::optional<at::Tensor>& draft,
                                                const at::Tensor& draft_tokens, const at::Tensor& row_indptr,
                                                const at::Tensor& accept_u, const at::Tensor& sample_u,
                                                const c10::optional<at::Tensor>& status);

}  // namespace mlora_torch
