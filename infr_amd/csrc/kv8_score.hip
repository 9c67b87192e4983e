// ScoreKv8: the attention weights each cached token has drawn, sum over the call's rows and the heads of its group
// of exp(score - lse). The scores are AttentionKv8's S^T = K Q^T again; V is not read.
//
// Few rows (at most 16 of a KV head): bound by reading the keys once. As in the attention a wave takes a page at a
// time; the 16 query rows' weights of a token are summed over the 16 lanes that hold them, each lane keeping one
// token at the end.
// Many rows: bound by the matrix cores and the exponential, 2 head_dim flops a pair, twice that in f16 products. A wave keeps a page's
// keys in registers as f16, four pages a workgroup, and 32 query rows at a time go through LDS, turned into hi + lo
// once for the four waves (two buffers, one barrier a step). Where pages are few, the rows are cut into parts whose
// sums a second kernel adds in their order, so that the same call gives the same bits.
// Measured: one token of 32 sequences of 1000 to 8000 tokens (8 KV heads of 128) 26 us, 4.6 TB/s; 1000 rows behind a
// prompt of 4001 tokens, 32 heads of 128, 4 KV heads, capped scores: 164 to 173 us, 170 TFLOP/s - by the kernel's counters
// vector instructions, the cap's series and the exponential above all, take 42 % of the time and matrix instructions 14 %; a
// compute unit has work for 59 % of it, since the first pages are seen by more rows than the last.
#include "kv8_attn.hpp"
#include "kv8_device.hpp"

namespace infr {

namespace {

// Adds the values of lanes l, l ^ 15 (^ 7, ^ 3, ^ 1) with DPP moves inside rows of 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
constexpr int kMirror = 0x140, kHalfMirror = 0x141, kQuadReverse = 0x1B, kQuadSwap = 0xB1;
// One step of the sum over 16 lanes: n values become n / 2, the half that bit `bit` of the lane names.
template <int CTRL, int N>
__device__ __forceinline__ void fold(float* x, bool upper) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
        const float mine = upper ? x[e + N / 2] : x[e], theirs = upper ? x[e] : x[e + N / 2];
        x[e] = mine + dpp<CTRL>(theirs);
    }
}

template <int DP, bool F8, bool GEN>
__global__ __launch_bounds__(64 * kStepWaves, DP <= 128 ? 2 : 1) void score_step_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a,
                                                                                       const float* __restrict__ lse,
                                                                                       float decay, int target, int whole) {
    constexpr int kCols = DP / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const SeqCut cut = find_cut(b, a, c.n_kv, kStepRows, target, whole, true, -1, (int)blockIdx.x);
    if (cut.s < 0 || !cut.q.ok) return;
    const int s = cut.s, parts = cut.parts, rest = (int)blockIdx.x - cut.first;
    const Kv8Seq q = cut.q;
    const SeqWork work = cut.work;
    const int part = rest % parts, h = rest / parts;
    const int per = (work.pages + parts - 1) / parts;
    const int p0 = part * per, p1 = min(p0 + per, (q.len + kPage - 1) / kPage);
    const bool live = col < q.n * a.group;
    const int i = live ? col / a.group : max(q.n - 1, 0), head = h * a.group + (live ? col % a.group : 0);

    const float cap = a.softcap * kLog2e, inv_cap = GEN ? inverse_cap(cap) : 0.0f;
    const bool use_pos = GEN && (a.window > 0 || a.slopes || a.first || a.prefix);
    const int all_see = a.causal ? q.len - q.n + 1 : q.len;
    const int32_t* table = b.pages + (size_t)s * b.max_pages;
    const int subs = kPage / c.block;
    uint4 kf[4][kCols];
    float ks = 0.0f;
    int page = 0, ids = 0, pos0 = 0;
    auto load_ids = [&](int p) {
        const int at = p + lane * kStepWaves;
        ids = at < p1 ? table[at] : 0;
        if (ids < 0 || ids >= c.n_pages) ids = -1;
    };
    auto load_keys = [&](int n) {
        page = __builtin_amdgcn_readlane(ids, n);
        const size_t at = (size_t)max(page, 0) * c.n_kv + h;
        const uint8_t* kp = c.k + at * (DP * kPage) + (16 * (col >> 2) + (col & 3)) * 64 + 16 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < kCols; ++j) kf[t][j] = load_stream(kp + j * kPage * 64 + t * 4 * 64);
        ks = c.ks[at * subs + g * 16 / c.block];
        if (use_pos) pos0 = c.pos[at * kPage];
    };
    int p = p0 + wave, n = 0;
    if (p < p1) {
        load_ids(p);
        load_keys(0);
    }
    __shared__ StepQ<DP, kStepRows> rows_q;
    stage_rows<DP, kStepRows>(rows_q, c, a, q, h, 0);
    __syncthreads();
    h8 qh[2 * kCols], ql[2 * kCols];
#pragma unroll
    for (int k = 0; k < 2 * kCols; ++k) {
        const int d = (k / 2) * 64 + g * 16 + (k % 2) * 8;
        qh[k] = *reinterpret_cast<const h8*>(&rows_q.x[col][d]);
        ql[k] = *reinterpret_cast<const h8*>(&rows_q.x[16 + col][d]);
    }
    const float row_factor = rows_q.factor[col];
    Kv8Row row{};
    row.window = a.window > 0 ? a.window : 0x7FFFFFFF;
    float row_lse = 0.0f;
    if (live) {
        row = kv8_row(b, a, q, s, i, head);
        row_lse = lse[(size_t)(q.r0 + i) * a.n_head + head] * kLog2e;
    }
    int last_pos = live ? row.pos : -0x7FFFFFFF - 1, last_first = live ? row.first : -0x7FFFFFFF - 1;
    if (use_pos)
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) {
            last_pos = max(last_pos, __shfl_xor(last_pos, k));
            last_first = max(last_first, __shfl_xor(last_first, k));
        }
    while (p < p1) {
        const int now = page;
        const size_t at = ((size_t)max(now, 0) * c.n_kv + h) * kPage + 16 * g;
        // (positions ascend: what the last row's window and document allow at the page's first token, all rows do)
        const bool masked = (p + 1) * kPage > min(all_see, q.len) || (use_pos && (last_pos - pos0 >= row.window || last_first > pos0));
        int kpos[16];
        if (use_pos && (masked || a.slopes)) {
            const int4* pp = reinterpret_cast<const int4*>(c.pos + at);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int4 x = pp[t];
                kpos[4 * t] = x.x, kpos[4 * t + 1] = x.y, kpos[4 * t + 2] = x.z, kpos[4 * t + 3] = x.w;
            }
        }
        const float old = decay != 0.0f ? c.sums[at + col] : 0.0f;
        f4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            sc[t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                const h8 lo = code_oct<F8>(kf[t][j].x, kf[t][j].y), hi = code_oct<F8>(kf[t][j].z, kf[t][j].w);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qh[2 * j], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qh[2 * j + 1], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, ql[2 * j], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ql[2 * j + 1], sc[t], 0, 0, 0);
            }
        }
        const int tok0 = p * kPage + 16 * g;
        const float factor = row_factor * ks;
        const int np = p + kStepWaves;
        if (np < p1) {
            if (++n == 64) {
                load_ids(np);
                n = 0;
            }
            load_keys(n);
        }
        float w[16];
        const bool bent = GEN && (a.softcap > 0.0f || a.slopes);
        float f = factor;
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = sc[e / 4][e % 4];
        if (bent) {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] *= factor;
            if (a.softcap > 0.0f) cap_scores<16, false>(w, cap, inv_cap);
            if (a.slopes)
#pragma unroll
                for (int e = 0; e < 16; ++e) w[e] = __builtin_fmaf(-row.slope, fabsf((float)(row.pos - kpos[e])), w[e]);
            f = 1.0f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(w[e], f, -row_lse));
            w[e] = live ? y : 0.0f;
        }
        if (masked)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int tok = tok0 + e;
                w[e] = tok < q.len && (use_pos ? row.sees(tok, kpos[e]) : tok <= row.slot) ? w[e] : 0.0f;
            }
        fold<kMirror, 16>(w, col & 8);
        fold<kHalfMirror, 8>(w, col & 4);
        fold<kQuadReverse, 4>(w, col & 2);
        fold<kQuadSwap, 2>(w, col & 1);
        if (now >= 0 && tok0 + col < q.len) c.sums[at + col] = (decay != 0.0f ? decay * old : 0.0f) + w[0];
        p = np;
    }
}

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 32;  // query rows of a step

// 32 query rows in LDS; rows are padded by 16 bytes.
template <int DP>
struct Rows {
    _Float16 hi[kTile][DP + 8], lo[kTile][DP + 8];
    float factor[kTile], lse[kTile], slope[kTile];
    int slot[kTile], pos[kTile], first[kTile];
    int last_first[kWaves];  // largest first[] of the rows each wave brought in
};

template <int DP, bool F8, bool GEN>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void score_prompt_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a,
                                                                                  const float* __restrict__ lse, float decay,
                                                                                  float* __restrict__ scratch, int parts) {
    constexpr int kSteps = DP / 16, kEach = DP / 8;  // a thread brings in kEach columns of a row: 8 threads a row
    extern __shared__ __align__(16) unsigned char smem[];
    Rows<DP>* rows = reinterpret_cast<Rows<DP>*>(smem);
    __shared__ __align__(16) int page_pos[kWaves][kPage];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, hf = lane >> 5;
    const int h = blockIdx.x / parts, part = blockIdx.x % parts, s = blockIdx.z;
    const Kv8Seq q = kv8_seq(b, s);
    const int n_pages = (q.len + kPage - 1) / kPage, group0 = (int)blockIdx.y * kWaves;
    if (!q.ok || group0 >= n_pages) return;
    const int p = group0 + wave;
    int page = p < n_pages ? b.pages[(size_t)s * b.max_pages + p] : -1;
    if (page < 0 || page >= c.n_pages) page = -1;
    const size_t at = (size_t)max(page, 0) * c.n_kv + h;
    const int subs = kPage / c.block;

    // the page's keys, A operands: MFMA row `col` is token my_tok of each half
    const int my_tok = (col & 3) + ((col >> 3) << 2) + (((col >> 2) & 1) << 4);
    h8 key[2][kSteps];
    float ks[2];
    const bool use_pos = GEN && (a.window > 0 || a.slopes || a.first || a.prefix);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        ks[t] = c.ks[at * subs + (32 * t + 16 * hf) / c.block];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const uint2 u = *reinterpret_cast<const uint2*>(c.k + at * (DP * kPage) + ((k / 4) * kPage + 32 * t + my_tok) * 64 + (k % 4) * 16 + hf * 8);
            key[t][k] = code_oct<F8>(u.x, u.y);
        }
    }
    if (use_pos) page_pos[wave][lane] = c.pos[at * kPage + lane];  // (the barrier before the first step comes in between)
    const int pos0 = use_pos ? c.pos[at * kPage] : 0;
    // rows that see any token of the workgroup's pages: by causality none before the first token's own, by the window
    // none from `window` behind the last one on (positions ascend strictly)
    const int t_first = group0 * kPage, t_last = min((group0 + kWaves) * kPage, q.len) - 1, begin = q.len - q.n;
    int i0 = 0, i1 = q.n;
    if (a.causal && !(a.prefix && a.prefix[s] > t_first)) i0 = max(i0, t_first - begin);
    if (a.window > 0) i1 = (int)min((int64_t)i1, (int64_t)t_last + a.window - begin);
    const int r_lo = i0 * a.group / kTile, r_hi = i1 > i0 ? (i1 * a.group + kTile - 1) / kTile : r_lo;
    const int per = (r_hi - r_lo + parts - 1) / parts;
    const int r0 = min(r_lo + part * per, r_hi), r1 = min(r0 + per, r_hi);

    const float cap = a.softcap * kLog2e, inv_cap = GEN ? inverse_cap(cap) : 0.0f;
    const int prefix = a.prefix ? a.prefix[s] : -0x7FFFFFFF - 1, window = a.window > 0 ? a.window : 0x7FFFFFFF;
    float v[kEach];
    Kv8Row in{};
    float in_lse = 0.0f;
    bool in_live = false;
    const int my_row = tid >> 3, my_col = (tid & 7) * kEach;
    const bool vec = rows_vec(c, a);
    auto fetch = [&](int rt) {
        const int rr = rt * kTile + my_row;
        in_live = rr < q.n * a.group;
        const int i = in_live ? rr / a.group : q.n - 1, head = h * a.group + (in_live ? rr % a.group : 0);
        const float* x = a.q + (size_t)(q.r0 + i) * a.q_stride + (size_t)head * c.dim;
        load_row<kEach>(x, my_col, c.dim, in_live, vec, v);
        in = kv8_row(b, a, q, s, i, head);
        in_lse = lse[(size_t)(q.r0 + i) * a.n_head + head] * kLog2e;
    };
    auto store = [&](Rows<DP>& r) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) top = max(top, abs_bits(v[e]));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        const int ex = row_exponent(top);
        const float down = a.scale < 0.0f ? -pow2(-ex) : pow2(-ex);
#pragma unroll
        for (int e = 0; e < kEach; e += 8) {
            h8 u, w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h2 hi, lo;
                split_pair(v[e + 2 * k] * down, v[e + 2 * k + 1] * down, &hi, &lo);
                u[2 * k] = hi[0], u[2 * k + 1] = hi[1];
                w[2 * k] = lo[0], w[2 * k + 1] = lo[1];
            }
            *reinterpret_cast<h8*>(&r.hi[my_row][my_col + e]) = u;
            *reinterpret_cast<h8*>(&r.lo[my_row][my_col + e]) = w;
        }
        if ((tid & 7) == 0) {
            r.factor[my_row] = fabsf(a.scale) * kLog2e * pow2(ex);
            r.lse[my_row] = in_lse;
            r.slope[my_row] = in.slope;
            r.slot[my_row] = in_live ? in.slot : -1;
            r.pos[my_row] = in.pos;
            r.first[my_row] = in_live ? in.first : 0x7FFFFFFF;
        }
        if (use_pos) {
            int most = in_live ? in.first : -0x7FFFFFFF - 1;
#pragma unroll
            for (int o = 8; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
            if (lane == 0) r.last_first[wave] = most;
        }
    };
    float acc[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) acc[e] = 0.0f;
    if (r0 < r1) {
        fetch(r0);
        store(rows[0]);
    }
    __syncthreads();
    for (int rt = r0; rt < r1; ++rt) {
        const Rows<DP>& r = rows[(rt - r0) & 1];
        const bool more = rt + 1 < r1;
        if (more) fetch(rt + 1);
        if (page >= 0) {
            f16x x[2];
            x[0] = (f16x)(0.0f);
            x[1] = (f16x)(0.0f);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const h8 hi = *reinterpret_cast<const h8*>(&r.hi[col][k * 16 + hf * 8]);
                const h8 lo = *reinterpret_cast<const h8*>(&r.lo[col][k * 16 + hf * 8]);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key[t][k], hi, x[t], 0, 0, 0);
                    x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key[t][k], lo, x[t], 0, 0, 0);
                }
            }
            const Kv8Row row{r.slot[col], r.pos[col], r.first[col], prefix, window, r.slope[col]};
            const float row_lse = r.lse[col];
            // tokens below this one are seen by all 32 rows (rows ascend, and so do their own tokens)
            const bool full = (rt + 1) * kTile <= q.n * a.group;
            const int all_see = a.causal ? begin + rt * kTile / a.group + 1 : q.len;
            bool masked = !full || (p + 1) * kPage > min(all_see, q.len);
            if (use_pos) {
                const int last_first = max(max(r.last_first[0], r.last_first[1]), max(r.last_first[2], r.last_first[3]));
                masked = masked || r.pos[kTile - 1] - pos0 >= window || last_first > pos0;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float factor = r.factor[col] * ks[t];
                if (GEN && (a.softcap > 0.0f || a.slopes)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[t][e] *= factor;
                    if (a.softcap > 0.0f) cap_scores<16, false>(x[t], cap, inv_cap);
                    if (a.slopes)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const int4 y = *reinterpret_cast<const int4*>(&page_pos[wave][32 * t + 16 * hf + e]);
                            const int kpos[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int n = 0; n < 4; ++n)
                                x[t][e + n] = __builtin_fmaf(-row.slope, fabsf((float)(row.pos - kpos[n])), x[t][e + n]);
                        }
                    factor = 1.0f;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) x[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][e], factor, -row_lse));
                if (masked)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        int4 y = make_int4(0, 0, 0, 0);
                        if (use_pos) y = *reinterpret_cast<const int4*>(&page_pos[wave][32 * t + 16 * hf + e]);
                        const int kpos[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const int tok = p * kPage + 32 * t + 16 * hf + e + n;
                            const bool yes = tok < q.len && row.first != 0x7FFFFFFF && (use_pos ? row.sees(tok, kpos[n]) : tok <= row.slot);
                            x[t][e + n] = yes ? x[t][e + n] : 0.0f;
                        }
                    }
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[16 * t + e] += x[t][e];
            }
        }
        if (more) store(rows[(rt + 1 - r0) & 1]);
        __syncthreads();
    }
    if (page < 0) return;
    // sum over the 32 lanes of a half: lane col ends with value `col` of acc, token 32 (col / 16) + 16 hf + col % 16
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float mine = col & 16 ? acc[e + 16] : acc[e], theirs = col & 16 ? acc[e] : acc[e + 16];
        acc[e] = mine + __shfl_xor(theirs, 16);
    }
    fold<kMirror, 16>(acc, col & 8);
    fold<kHalfMirror, 8>(acc, col & 4);
    fold<kQuadReverse, 4>(acc, col & 2);
    fold<kQuadSwap, 2>(acc, col & 1);
    const int t = 32 * (col >> 4) + 16 * hf + (col & 15);
    if (p * kPage + t >= q.len) return;
    if (parts > 1) {
        scratch[((((size_t)s * b.max_pages + p) * c.n_kv + h) * parts + part) * kPage + t] = acc[0];
        return;
    }
    float* out = c.sums + at * kPage + t;
    *out = (decay != 0.0f ? decay * *out : 0.0f) + acc[0];
}

// Adds the parts of one page's sums, in their order: a wave per (page, head).
__global__ __launch_bounds__(64) void score_join_kernel(Kv8Cache c, Kv8Batch b, float decay, const float* __restrict__ scratch, int parts) {
    const int s = blockIdx.z, h = blockIdx.x, p = blockIdx.y, t = threadIdx.x;
    const Kv8Seq q = kv8_seq(b, s);
    if (!q.ok || p * kPage + t >= q.len) return;
    const int page = b.pages[(size_t)s * b.max_pages + p];
    if (page < 0 || page >= c.n_pages) return;
    const float* from = scratch + (((size_t)s * b.max_pages + p) * c.n_kv + h) * parts * kPage + t;
    float x = 0.0f;
    for (int k = 0; k < parts; ++k) x += from[(size_t)k * kPage];
    float* out = c.sums + ((size_t)page * c.n_kv + h) * kPage + t;
    *out = (decay != 0.0f ? decay * *out : 0.0f) + x;
}

// The form for few rows has one column tile.
bool few_rows(int max_q, int group) { return (int64_t)max_q * group <= kStepRows; }

// Parts of the rows: enough workgroups for two on each compute unit, four steps of rows at least in a part. The workgroups
// are counted by the page table's width: a table far wider than the sequences are long leaves the rows in one part (1000 rows
// behind 4001 tokens, 64 / 2048 pages: 166 / 720 us).
int parts_of(int cus, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    const int64_t wgs = (int64_t)n_seq * n_kv * ((max_pages + kWaves - 1) / kWaves);
    const int64_t steps = ((int64_t)max_q * group + kTile - 1) / kTile;
    return (int)std::max<int64_t>(1, std::min<int64_t>(2 * cus / wgs, steps / 4));
}

template <int DP>
void launch_score_dp(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, const float* lse, float decay, float* scratch,
                     int cus, hipStream_t stream) {
    const bool gen = a.softcap > 0.0f || a.window > 0 || a.slopes || a.first || a.prefix;
    if (few_rows(b.max_q, a.group)) {
        auto kernel = c.f8 ? (gen ? score_step_kernel<DP, true, true> : score_step_kernel<DP, true, false>)
                           : (gen ? score_step_kernel<DP, false, true> : score_step_kernel<DP, false, false>);
        // pieces: there is no join here, so no sequence has to be whole, and three for each compute unit level out best
        // (32 sequences' step: 27 us; two or four 29)
        const int64_t heads = (int64_t)b.n_seq * c.n_kv;
        const int target = 3 * cus;
        const unsigned items = (unsigned)std::min(target + heads, heads * ((b.max_pages + kStepWaves - 1) / kStepWaves));
        hipLaunchKernelGGL(kernel, dim3(items), dim3(64 * kStepWaves), 0, stream, c, b, a, lse, decay, target, kStepWaves);
        return;
    }
    const int parts = parts_of(cus, c.n_kv, a.group, b.n_seq, b.max_q, b.max_pages);
    auto kernel = c.f8 ? (gen ? score_prompt_kernel<DP, true, true> : score_prompt_kernel<DP, true, false>)
                       : (gen ? score_prompt_kernel<DP, false, true> : score_prompt_kernel<DP, false, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(c.n_kv * parts), (unsigned)((b.max_pages + kWaves - 1) / kWaves), (unsigned)b.n_seq),
                       dim3(kThreads), 2 * sizeof(Rows<DP>), stream, c, b, a, lse, decay, scratch, parts);
    if (parts > 1)
        hipLaunchKernelGGL(score_join_kernel, dim3((unsigned)c.n_kv, (unsigned)b.max_pages, (unsigned)b.n_seq), dim3(64), 0, stream,
                           c, b, decay, scratch, parts);
}

}  // namespace

size_t score_kv8_scratch(int cus, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    if (few_rows(max_q, group)) return 0;
    const int parts = parts_of(cus, n_kv, group, n_seq, max_q, max_pages);
    return parts == 1 ? 0 : (size_t)n_seq * max_pages * n_kv * parts * kPage * sizeof(float);
}

void launch_score_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, const float* lse, float decay, void* scratch, int cus,
                      hipStream_t stream) {
    float* f = static_cast<float*>(scratch);
    switch (c.dp) {
    case 64: launch_score_dp<64>(c, b, a, lse, decay, f, cus, stream); break;
    case 128: launch_score_dp<128>(c, b, a, lse, decay, f, cus, stream); break;
    case 192: launch_score_dp<192>(c, b, a, lse, decay, f, cus, stream); break;
    default: launch_score_dp<256>(c, b, a, lse, decay, f, cus, stream); break;
    }
}

}  // namespace infr
