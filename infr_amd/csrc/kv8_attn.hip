// AttentionKv8 and ScoreKv8, one wave per query row and head: lane t holds token t of a page.
#include "kv8_attn.hpp"

namespace infr {

namespace {

struct RowSees {
    int len, slot, pos, first, prefix, window;
    bool causal;
    __device__ __forceinline__ bool operator()(int j, int kpos) const {
        return j < len && (!causal || j <= slot || kpos < prefix) && (window == 0 || pos - kpos < window) && kpos >= first;
    }
};

__device__ __forceinline__ RowSees row_sees(const Kv8Batch& b, const Kv8Attn& a, const Kv8Seq& q, int s, int i) {
    RowSees r;
    r.len = q.len;
    r.slot = q.len - q.n + i;
    r.pos = b.pos[q.r0 + i];
    r.first = a.first ? a.first[q.r0 + i] : -0x7FFFFFFF - 1;
    r.prefix = a.prefix ? a.prefix[s] : -0x7FFFFFFF - 1;
    r.window = a.window;
    r.causal = a.causal != 0;
    return r;
}

__device__ __forceinline__ float score_of(const Kv8Attn& a, float dot, int head, int pos, int kpos) {
    float s = a.scale * dot;
    if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
    if (a.slopes) s -= a.slopes[head] * fabsf((float)(pos - kpos));
    return s;
}

__device__ __forceinline__ float dot_of(const Kv8Cache& c, const float* q, int page, int h, int t) {
    float acc = 0.0f;
    for (int d = 0; d < c.dim; ++d) acc = __builtin_fmaf(q[d], kv8_value(c.k[k_at(c, page, h, t, d)], c.f8 != 0), acc);
    return acc * c.ks[((size_t)page * c.n_kv + h) * (kPage / c.block) + t / c.block];
}

__global__ __launch_bounds__(64) void score_rows_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a, const float* __restrict__ lse,
                                                        float decay) {
    const int s = blockIdx.z, h = blockIdx.y, p = blockIdx.x, lane = threadIdx.x;
    const Kv8Seq q = kv8_seq(b, s);
    if (!q.ok || p * kPage >= q.len) return;
    const int page = b.pages[(size_t)s * b.max_pages + p];
    if (page < 0 || page >= c.n_pages) return;
    const size_t at = ((size_t)page * c.n_kv + h) * kPage + lane;
    const int kpos = c.pos[at], j = p * kPage + lane;
    float acc = 0.0f;
    for (int i = 0; i < q.n; ++i) {
        const RowSees sees = row_sees(b, a, q, s, i);
        if (!sees(j, kpos)) continue;
        for (int g = 0; g < a.group; ++g) {
            const int head = h * a.group + g;
            const float x = score_of(a, dot_of(c, a.q + (size_t)(q.r0 + i) * a.q_stride + (size_t)head * c.dim, page, h, lane),
                                     head, sees.pos, kpos);
            acc += expf(x - lse[(size_t)(q.r0 + i) * a.n_head + head]);
        }
    }
    if (j < q.len) c.sums[at] = (decay == 0.0f ? 0.0f : decay * c.sums[at]) + acc;
}

}  // namespace

size_t attention_kv8_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    if (prompt_takes(max_q, group)) return prompt_scratch(cus, dim, n_kv, group, n_seq, max_q, max_pages);
    return step_scratch(cus, dim, n_kv, group, n_seq, max_q, max_pages);
}

void launch_attention_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, void* scratch, int cus,
                          hipStream_t stream) {
    if (prompt_takes(b.max_q, a.group)) launch_attention_prompt(c, b, a, dst, lse, static_cast<float*>(scratch), cus, stream);
    else launch_attention_step(c, b, a, dst, lse, static_cast<float*>(scratch), cus, stream);
}

void launch_score_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, const float* lse, float decay,
                      hipStream_t stream) {
    hipLaunchKernelGGL(score_rows_kernel, dim3((unsigned)b.max_pages, (unsigned)c.n_kv, (unsigned)b.n_seq), dim3(64), 0,
                       stream, c, b, a, lse, decay);
}

}  // namespace infr
