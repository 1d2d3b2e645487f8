// Operators of torch_ops.cpp that torch_direct.cpp calls as well.
#pragma once
#include <ATen/ATen.h>

#include <optional>
#include <tuple>

namespace fdl_torch {

using Scores = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

void page_slots(const at::Tensor& lens, const at::Tensor& n_new, const at::Tensor& block_table,
                const at::Tensor& free_pages, const at::Tensor& free_count, int64_t page_size,
                const at::Tensor& slots, const at::Tensor& positions, const at::Tensor& cu_seqlens,
                const std::optional<at::Tensor>& new_lens, const std::optional<at::Tensor>& new_count);
void norm_rope_store(const at::Tensor& y, const at::Tensor& positions, const at::Tensor& inv_freq,
                     const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight, double eps,
                     bool interleaved, double rope_scale, const at::Tensor& q, const at::Tensor& k_pages,
                     const at::Tensor& v_pages, const at::Tensor& slots);
void paged_decode_attn(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
                       const at::Tensor& block_table, const at::Tensor& lens, double scale, const at::Tensor& out);
Scores token_logprobs(const at::Tensor& logits, const at::Tensor& targets, int64_t top, bool one);

}  // namespace fdl_torch
