// Host entry points of the tree-drafted decoding operators (bound in bindings.cpp).
#pragma once
#include <torch/extension.h>

namespace kvs {

void plan_step(torch::Tensor ctx_lens, torch::Tensor new_lens, torch::Tensor block_tables, torch::Tensor held,
               torch::Tensor free_queue, torch::Tensor cursor, int64_t block_size,
               c10::optional<torch::Tensor> parents, torch::Tensor indptr, torch::Tensor row_request,
               torch::Tensor positions, torch::Tensor slot_mapping, c10::optional<torch::Tensor> tree_mask,
               torch::Tensor held_out, torch::Tensor cursor_out, torch::Tensor status);
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
void commit_tree(torch::Tensor draft_ids, torch::Tensor target_ids, c10::optional<torch::Tensor> parents,
                 torch::Tensor indptr, torch::Tensor ctx_lens, torch::Tensor slot_mapping,
                 c10::optional<torch::Tensor> tree_kv, c10::optional<torch::Tensor> kv_cache,
                 c10::optional<torch::Tensor> tokens, torch::Tensor accepted, torch::Tensor path,
                 torch::Tensor next_ids, torch::Tensor ctx_out, torch::Tensor status);

}  // namespace kvs
