// AttentionKv8: which of its forms a call takes.
#include "kv8_attn.hpp"

namespace infr {

size_t attention_kv8_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    if (prompt_takes(max_q, group)) return prompt_scratch(cus, dim, n_kv, group, n_seq, max_q, max_pages);
    return step_scratch(cus, dim, n_kv, group, n_seq, max_q, max_pages);
}

void launch_attention_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, void* scratch, int cus,
                          hipStream_t stream) {
    if (prompt_takes(b.max_q, a.group)) launch_attention_prompt(c, b, a, dst, lse, static_cast<float*>(scratch), cus, stream);
    else launch_attention_step(c, b, a, dst, lse, static_cast<float*>(scratch), cus, stream);
}

}  // namespace infr
