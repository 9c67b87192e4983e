// The two forms of AttentionKv8: few rows per sequence (kv8_step.hip) and many (kv8_prompt.hip).
#pragma once

#include <algorithm>

#include "kv8.hpp"

namespace infr {

size_t step_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages);
void launch_attention_step(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch,
                           int cus, hipStream_t stream);

size_t prompt_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages);
void launch_attention_prompt(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch,
                             int cus, hipStream_t stream);

}  // namespace infr
