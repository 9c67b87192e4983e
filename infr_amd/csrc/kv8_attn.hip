// AttentionKv8 and ScoreKv8, one wave per query row and head: lane t holds token t of a page.
#include "kv8.hpp"

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

__global__ __launch_bounds__(64) void attention_rows_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a, float* __restrict__ dst,
                                                            float* __restrict__ lse) {
    const int s = blockIdx.z, head = blockIdx.y, i = blockIdx.x, lane = threadIdx.x, h = head / a.group;
    const Kv8Seq q = kv8_seq(b, s);
    if (i >= q.n) return;
    float* out = dst + ((size_t)(q.r0 + i) * a.n_head + head) * c.dim;
    const float* qr = a.q + (size_t)(q.r0 + i) * a.q_stride + (size_t)head * c.dim;
    float o[4] = {0, 0, 0, 0}, m = -__builtin_inff(), l = 0.0f;
    bool bad = !q.ok;
    if (q.ok) {
        const RowSees sees = row_sees(b, a, q, s, i);
        for (int p = 0; p * kPage < q.len; ++p) {
            const int page = b.pages[(size_t)s * b.max_pages + p];
            if (page < 0 || page >= c.n_pages) {
                bad = true;
                break;
            }
            const int j = p * kPage + lane;
            const int kpos = c.pos[((size_t)page * c.n_kv + h) * kPage + lane];
            const bool see = sees(j, kpos);
            const float x = see ? score_of(a, dot_of(c, qr, page, h, lane), head, sees.pos, kpos) : -__builtin_inff();
            float top = x;
            bool nan = see && x != x;
            for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
            if (__ballot(nan)) bad = true;
            if (!__ballot(see)) continue;
            const float m2 = fmaxf(m, top), keep = expf(m - m2);
            const float w = see ? expf(x - m2) : 0.0f;
            float sum = w;
            for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
            l = l * keep + sum;
            m = m2;
            for (int e = 0; e < 4; ++e) {
                const int d = e * 64 + lane;
                o[e] *= keep;
                for (int t = 0; t < 64; ++t) {
                    const float wt = __shfl(w, t);
                    if (wt == 0.0f || d >= c.dim) continue;
                    const float vs = c.vs[((size_t)page * c.n_kv + h) * (kPage / c.block) + t / c.block];
                    o[e] = __builtin_fmaf(wt, kv8_value(c.v[v_at(c, page, h, t, d)], c.f8 != 0) * vs, o[e]);
                }
            }
        }
    }
    for (int e = 0; e < 4; ++e)
        if (e * 64 + lane < c.dim) out[e * 64 + lane] = bad ? __builtin_nanf("") : l > 0.0f ? o[e] / l : l == 0.0f ? 0.0f : l;
    if (lse && lane == 0) lse[(size_t)(q.r0 + i) * a.n_head + head] = bad ? __builtin_nanf("") : m + logf(l);
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

size_t attention_kv8_scratch(int, int, int, int, int, int) { return 0; }

void launch_attention_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, void*,
                          hipStream_t stream) {
    hipLaunchKernelGGL(attention_rows_kernel, dim3((unsigned)b.max_q, (unsigned)a.n_head, (unsigned)b.n_seq), dim3(64), 0,
                       stream, c, b, a, dst, lse);
}

void launch_score_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, const float* lse, float decay,
                      hipStream_t stream) {
    hipLaunchKernelGGL(score_rows_kernel, dim3((unsigned)b.max_pages, (unsigned)c.n_kv, (unsigned)b.n_seq), dim3(64), 0,
                       stream, c, b, a, lse, decay);
}

}  // namespace infr
