// Host entry points of the tree-drafted decoding operators (bound in bindings.cpp).
#pragma once
#include <torch/extension.h>

#include <vector>

namespace kvs {

// Outputs [indptr, row_request, positions, slot_mapping, (tree_mask), held, cursor]; `out` may give them.
std::vector<torch::Tensor> plan_step(torch::Tensor ctx_lens, torch::Tensor new_lens, torch::Tensor block_tables,
                                     torch::Tensor held, torch::Tensor free_queue, torch::Tensor cursor,
                                     int64_t block_size, int64_t num_rows, c10::optional<torch::Tensor> parents,
                                     int64_t max_tree, std::vector<torch::Tensor> out, torch::Tensor status);
void paged_tree_attention(torch::Tensor q, torch::Tensor k_tree, torch::Tensor v_tree, torch::Tensor k_cache,
                          torch::Tensor v_cache, torch::Tensor block_tables, torch::Tensor ctx_lens,
                          torch::Tensor indptr, c10::optional<torch::Tensor> tree_mask, double scale,
                          torch::Tensor out, torch::Tensor status);
void process_logits(torch::Tensor logits, torch::Tensor out, c10::optional<torch::Tensor> row_request,
                    c10::optional<torch::Tensor> tokens, c10::optional<torch::Tensor> token_lens,
                    c10::optional<torch::Tensor> prompt_lens, c10::optional<torch::Tensor> repetition,
                    c10::optional<torch::Tensor> frequency, c10::optional<torch::Tensor> presence,
                    c10::optional<torch::Tensor> bias_ids, c10::optional<torch::Tensor> bias_values,
                    c10::optional<torch::Tensor> allowed, c10::optional<torch::Tensor> allowed_index,
                    c10::optional<torch::Tensor> draft_ids, c10::optional<torch::Tensor> indptr,
                    c10::optional<torch::Tensor> tree_mask, c10::optional<torch::Tensor> positions,
                    int64_t vocab_begin, c10::optional<torch::Tensor> greedy, c10::optional<torch::Tensor> greedy_val);
// Outputs [accepted, path, next_ids, ctx_lens]; `out` may give them.
std::vector<torch::Tensor> commit_tree(torch::Tensor draft_ids, torch::Tensor target_ids,
                                       c10::optional<torch::Tensor> parents, torch::Tensor indptr,
                                       torch::Tensor ctx_lens, torch::Tensor slot_mapping,
                                       c10::optional<torch::Tensor> tree_kv, c10::optional<torch::Tensor> kv_cache,
                                       c10::optional<torch::Tensor> tokens, std::vector<torch::Tensor> out,
                                       torch::Tensor status);

}  // namespace kvs
