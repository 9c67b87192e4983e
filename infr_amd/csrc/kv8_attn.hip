// AttentionKv8: which of its forms a call takes.
#include "kv8_attn.hpp"

namespace infr {

namespace {

// Whether the form for many rows takes this shape. It needs some 20 us for the smallest call, a workgroup going through
// a tile's pages in turn; the form for few rows cuts them up, but reads a page again for every 16 rows. So up to 32 rows
// of a KV head the latter, and up to 256 as long as its tiles are no more than two for a compute unit, and their pages 32
// (8 KV heads of 128, few / many: 64 rows behind 3000 tokens 15 / 28 us, behind 16000 33 / 42, 256 behind 3000 25 / 31,
// 128 of each of 4 sequences of 600 to 1000 20 / 26, a prompt of 60 tokens, 4 heads to each, 8.0 / 10.1; but 64 of each of
// 8 sequences of 500 to 8000 49 / 44, and three packed prompts of 250 tokens, 16 heads, 22 / 16). Pages are counted by the page table's
// width: with a table of 2048 pages the prompt of 60 tokens takes 28 us, the 256 rows behind 3000 tokens 36.
bool prompt_takes(int cus, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    const int64_t rows = (int64_t)max_q * group, tiles = (rows + 15) / 16 * n_seq * n_kv;
    return rows > 32 && (rows > 256 || tiles > (int64_t)2 * cus || tiles * max_pages > (int64_t)32 * cus);
}

}  // namespace

size_t attention_kv8_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    if (prompt_takes(cus, n_kv, group, n_seq, max_q, max_pages)) return prompt_scratch(cus, dim, n_kv, group, n_seq, max_q, max_pages);
    return step_scratch(cus, dim, n_kv, group, n_seq, max_q, max_pages);
}

void launch_attention_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, void* scratch, int cus,
                          hipStream_t stream) {
    if (prompt_takes(cus, c.n_kv, a.group, b.n_seq, b.max_q, b.max_pages)) launch_attention_prompt(c, b, a, dst, lse, static_cast<float*>(scratch), cus, stream);
    else launch_attention_step(c, b, a, dst, lse, static_cast<float*>(scratch), cus, stream);
}

}  // namespace infr
