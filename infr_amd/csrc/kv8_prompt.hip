// AttentionKv8 for many rows per sequence: prompts and their chunks. Bound by the matrix cores: 4 head_dim flops for
// each pair of row and key that see each other, twice that in f16 products (hi + lo).
//
// A workgroup takes 128 query rows of one (sequence, KV head) - tokens times the heads of the group, so that a page
// of keys serves the whole group - and walks over the pages; each of its four waves owns 32 rows, the columns of the
// 32x32x16 f16 MFMA. The page's codes become f16 once per workgroup on their way into LDS (two buffers: the next
// page's codes are requested before the current page is multiplied and written behind it, one barrier a page); a
// wave's scores, softmax and output stay in its registers. Tokens are dealt to the MFMA's rows so that a lane holds
// 16 neighbours: one block's scale, and P.V's operand as it stands.
// Measured: 4096 tokens, 32 heads of 128, 8 KV heads: 278 us one call behind the other for 0.15 s, 495 TFLOP/s, twice that
// in f16 products (a large f16 product of the library: 1260); the kernel alone in short bursts, on a card less warmed up,
// 299 to 328. By its counters there, at 1.96 GHz, matrix instructions take 45 % of the time and vector instructions 46 %,
// and a third of either overlaps. Three packed prompts of 700 to 2501 tokens, 16 heads of 80: 63 to 77 us by the machine,
// 11 % matrix and 35 % vector instructions: a tile's pages follow one another, and between them it waits.
// With few row tiles a workgroup takes 64 rows instead, two waves to 32 of them, each with half of every page's tokens, and
// joins their results in LDS at the end.
// Pages no row of the workgroup sees are not visited; pages all rows of a wave see take no mask.
#include "kv8_attn.hpp"
#include "kv8_device.hpp"

namespace infr {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 32;                // query rows of a wave

// Waves that share 32 query rows, each with 64 / KS tokens of every page; rows of a workgroup.
template <int KS>
constexpr int kRows = kCols * kWaves / KS;
template <int DP, int KS>
constexpr int kPieceFloats = kRows<KS> * DP + 2 * kRows<KS>;

// A page's first DC columns in LDS. Rows are padded by 16 bytes: neighbours then start four banks apart.
template <int DC>
struct Stage {
    _Float16 k[kPage][DC + 8];
    _Float16 v[DC][kPage + 8];
    float ks[4], vs[4];    // scales of the four runs of 16 tokens
    int32_t pos[kPage];
};

// DC: the columns that are computed with, head_dim rounded up to 32.
template <int DP, int DC, int KS, bool F8, bool GEN>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void prompt_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a,
                                                                            float* __restrict__ dst, float* __restrict__ lse,
                                                                            float* __restrict__ scratch, int tiles, int parts) {
    constexpr int kSteps = DC / 16;  // of the scores' sum
    constexpr int kOut = DC / 32;    // output tiles
    constexpr int kLoads = DP / 64;  // 16-byte pieces of K, and of V, that a thread brings in
    constexpr int kHalves = 2 / KS;  // of a page that a wave takes
    constexpr int kRows = infr::kRows<KS>;
    extern __shared__ __align__(16) unsigned char smem[];
    Stage<DC>* stage = reinterpret_cast<Stage<DC>*>(smem);
    __shared__ int first_page[kWaves], last_page[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, hf = lane >> 5;
    const int h = blockIdx.x / parts, part = blockIdx.x % parts, s = blockIdx.y;
    const int rt = tiles - 1 - (int)blockIdx.z;  // causal rows get longer: the long ones of all sequences start first
    const Kv8Seq q = kv8_seq(b, s);
    const int n_rows = q.n * a.group;
    if (rt * kRows >= n_rows) return;
    const int half0 = KS == 2 ? wave & 1 : 0;  // first of the wave's halves
    const int rr = rt * kRows + wave / KS * kCols + col;
    const bool live = rr < n_rows;
    const int i = live ? rr / a.group : q.n - 1, head = h * a.group + (live ? rr % a.group : 0);
    const Kv8Row row = kv8_row(b, a, q, s, i, head);

    // Tokens the row can see at all lie in [lo, hi): positions ascend strictly and are not negative, so a token is at
    // least as far from the row in positions as in tokens, and none with a position below `prefix` lies behind it. A
    // document that begins behind the row has none of the tokens up to the row's own; one that begins at 0 or before has
    // all there are (and a distance to it may not fit an int).
    int lo = 0x7FFFFFFF, hi = 0;
    if (live && q.ok) {
        const int slot = q.len - q.n + i;
        lo = 0;
        if (a.window > 0) lo = max(lo, slot - a.window + 1);
        if (a.first && row.first > 0) lo = max(lo, row.pos >= row.first ? slot - (row.pos - row.first) : slot + 1);
        hi = a.causal ? max(slot + 1, min(a.prefix ? row.prefix : 0, q.len)) : q.len;
    }
    int last_pos = live ? row.pos : -0x7FFFFFFF - 1, last_first = live ? row.first : -0x7FFFFFFF - 1;
    int full_hi = live ? (a.causal ? q.len - q.n + i + 1 : q.len) : 0x7FFFFFFF;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
        full_hi = min(full_hi, __shfl_xor(full_hi, o));
        last_pos = max(last_pos, __shfl_xor(last_pos, o));
        last_first = max(last_first, __shfl_xor(last_first, o));
    }
    // this wave's pages; none when lo >= hi
    const int w0 = lo < hi ? lo / kPage : 0x7FFFFFFF, w1 = lo < hi ? (hi + kPage - 1) / kPage : 0;
    if (lane == 0) {
        first_page[wave] = w0;
        last_page[wave] = w1;
    }
    __syncthreads();
    int g0 = 0x7FFFFFFF, g1 = 0;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        g0 = min(g0, first_page[k]);
        g1 = max(g1, last_page[k]);
    }
    int p0 = min(g0, g1), p1 = g1;
    if (parts > 1) {
        const int per = (p1 - p0 + parts - 1) / parts;
        p0 = min(p0 + part * per, p1);
        p1 = min(p0 + per, p1);
    }

    h8 qh[kSteps], ql[kSteps];
    float row_factor;
    {
        const float* x = a.q + (size_t)(q.r0 + i) * a.q_stride + (size_t)head * c.dim;
        const bool vec = rows_vec(c, a);
        float v[kSteps][8];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            load_row<8>(x, k * 16 + hf * 8, c.dim, live, vec, v[k]);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[k][e]));
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const int e2 = row_exponent(top);
        const float down = a.scale < 0.0f ? -pow2(-e2) : pow2(-e2);  // factors stay positive: a maximum may be taken before them
        row_factor = fabsf(a.scale) * kLog2e * pow2(e2);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                h2 u, w;
                split_pair(v[k][2 * o] * down, v[k][2 * o + 1] * down, &u, &w);
                qh[k][2 * o] = u[0], qh[k][2 * o + 1] = u[1];
                ql[k][2 * o] = w[0], ql[k][2 * o + 1] = w[1];
            }
        }
    }
    const float cap = a.softcap * kLog2e, inv_cap = GEN ? inverse_cap(cap) : 0.0f;
    const bool use_pos = GEN && (a.window > 0 || a.slopes || a.first || a.prefix);

    f16x o[kOut];
#pragma unroll
    for (int k = 0; k < kOut; ++k) o[k] = (f16x)(0.0f);
    float top = kNoMax, sum = 0.0f;
    float v_exp = kNoExp;  // O's unit: 2^v_exp / 2^kBias
    bool bad = !q.ok, v_bad = false;  // v_bad: the row sees a token whose value is NaN

    const int32_t* table = b.pages + (size_t)s * b.max_pages;
    const int subs = kPage / c.block;
    // codes of one page on their way: thread -> token / column tid / 4, 16 bytes tid % 4 of each 64
    uint4 kr[kLoads], vr[kLoads];
    float sr = 0.0f;
    int pr = 0;
    auto fetch = [&](int p) {
        int page = table[p];
        if (page < 0 || page >= c.n_pages) {
            bad = true;
            page = 0;
        }
        const size_t at = (size_t)page * c.n_kv + h;
        const uint8_t* kp = c.k + at * (DP * kPage) + tid * 16;
        const uint8_t* vp = c.v + at * (DP * kPage) + tid * 16;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            if ((j + 1) * 64 <= DC || (tid & 3) < 2) kr[j] = *reinterpret_cast<const uint4*>(kp + j * kThreads * 16);
            if ((j + 1) * 64 <= DC || tid < 128) vr[j] = *reinterpret_cast<const uint4*>(vp + j * kThreads * 16);
        }
        if (tid < 8) sr = (tid < 4 ? c.ks : c.vs)[at * subs + (tid & 3) * 16 / c.block];
        if (use_pos && tid < kPage) pr = c.pos[at * kPage + tid];
        if (F8 && (p + 1) * kPage > q.len) {  // what stands behind the last token may be NaN as a code
            const int left = min(max(q.len - p * kPage - (tid & 3) * 16, 0), 16);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                uint32_t* u = reinterpret_cast<uint32_t*>(&vr[j]);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int m = min(max(left - 4 * t, 0), 4);
                    u[t] = m == 4 ? u[t] : u[t] & ((1u << (8 * m)) - 1u);
                }
            }
        }
    };
    auto store = [&](Stage<DC>& st) {
        const int t = tid >> 2, e = (tid & 3) * 16;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            if ((j + 1) * 64 <= DC || e < 32) {
                *reinterpret_cast<h8*>(&st.k[t][j * 64 + e]) = code_oct<F8>(kr[j].x, kr[j].y);
                *reinterpret_cast<h8*>(&st.k[t][j * 64 + e + 8]) = code_oct<F8>(kr[j].z, kr[j].w);
            }
            if ((j + 1) * 64 <= DC || t < 32) {
                *reinterpret_cast<h8*>(&st.v[j * 64 + t][e]) = code_oct<F8>(vr[j].x, vr[j].y);
                *reinterpret_cast<h8*>(&st.v[j * 64 + t][e + 8]) = code_oct<F8>(vr[j].z, vr[j].w);
            }
        }
        if (tid < 4) st.ks[tid] = sr;
        else if (tid < 8) st.vs[tid - 4] = sr;
        if (use_pos && tid < kPage) st.pos[tid] = pr;
    };

    if (p0 < p1) {
        fetch(p0);
        store(stage[0]);
    }
    __syncthreads();
    const int my_tok = (col & 3) + ((col >> 3) << 2) + (((col >> 2) & 1) << 4);  // token of MFMA row `col`
    for (int p = p0; p < p1; ++p) {
        const Stage<DC>& st = stage[(p - p0) & 1];
        const bool more = p + 1 < p1;
        if (more) fetch(p + 1);
        if (p >= w0 && p < w1) {
            // x[t][e]: token 32 (half0 + t) + 16 hf + e of the page
            f16x x[kHalves];
#pragma unroll
            for (int t = 0; t < kHalves; ++t) x[t] = (f16x)(0.0f);
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int t = 0; t < kHalves; ++t) {
                    const h8 key = *reinterpret_cast<const h8*>(&st.k[(half0 + t) * 32 + my_tok][k * 16 + hf * 8]);
                    x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, qh[k], x[t], 0, 0, 0);
                    x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, ql[k], x[t], 0, 0, 0);
                }
            // (positions ascend: what the last row's window and document allow at the page's first token, all rows allow)
            const bool masked = (p + 1) * kPage > min(full_hi, q.len) ||
                                (use_pos && (last_pos - st.pos[0] >= row.window || last_first > st.pos[0]));
            const bool bent = GEN && (a.softcap > 0.0f || a.slopes);
            float high = -__builtin_inff(), factor[kHalves], vs[kHalves], highs[kHalves];
            bool any[kHalves];
#pragma unroll
            for (int t = 0; t < kHalves; ++t) {
                factor[t] = row_factor * st.ks[2 * (half0 + t) + hf];
                vs[t] = st.vs[2 * (half0 + t) + hf];
                any[t] = true;
                if (masked || bent) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[t][e] *= factor[t];
                    if (GEN && a.softcap > 0.0f) cap_scores<16, true>(x[t], cap, inv_cap);
                    factor[t] = 1.0f;
                }
                if (GEN && a.slopes)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int4 y = *reinterpret_cast<const int4*>(&st.pos[(half0 + t) * 32 + hf * 16 + e]);
                        const int kpos[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int n = 0; n < 4; ++n)  // (the difference is taken in integers: positions may be any)
                            x[t][e + n] = __builtin_fmaf(-row.slope, fabsf((float)(row.pos - kpos[n])), x[t][e + n]);
                    }
                if (masked) {
                    const int tok0 = p * kPage + (half0 + t) * 32 + hf * 16;
                    any[t] = false;
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        int4 y = make_int4(0, 0, 0, 0);
                        if (use_pos) y = *reinterpret_cast<const int4*>(&st.pos[(half0 + t) * 32 + hf * 16 + e]);
                        const int kpos[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const int tok = tok0 + e + n;
                            const bool yes = tok < q.len && (use_pos ? row.sees(tok, kpos[n]) : tok <= row.slot);
                            any[t] = any[t] || yes;
                            x[t][e + n] = yes ? x[t][e + n] : -__builtin_inff();
                        }
                    }
                }
                float most = x[t][0];
#pragma unroll
                for (int e = 1; e < 16; ++e) most = fmaxf(most, x[t][e]);
                highs[t] = most * factor[t];
                high = fmaxf(high, highs[t]);
            }
            if (__any(fabsf(high) > kLargeScore))
#pragma unroll
                for (int t = 0; t < kHalves; ++t) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[t][e] *= factor[t];
                    factor[t] = 1.0f;
                }
            auto product = [&](float over) {
                float e = product_exponent(vs[0], highs[0], over);
                if (kHalves == 2) e = fmaxf(e, product_exponent(vs[kHalves - 1], highs[kHalves - 1], over));
                return e;
            };
            if (__any(high > top + kLag || product(top) > v_exp + kLag)) {
                const float new_top = fmaxf(top, halves_max(high)), down = top - new_top;
                const float new_exp = fmaxf(fmaxf(__builtin_ceilf(v_exp + down), __builtin_ceilf(halves_max(product(new_top)))), kNoExp);
                const float keep_o = __builtin_amdgcn_exp2f(v_exp + down - new_exp);
                sum *= __builtin_amdgcn_exp2f(down);
#pragma unroll
                for (int k = 0; k < kOut; ++k) o[k] *= keep_o;
                top = new_top;
                v_exp = new_exp;
            }
            // weights times the values' scale in one exponential; their sum is divided by it
            h8 wh[2 * kHalves], wl[2 * kHalves];
#pragma unroll
            for (int t = 0; t < kHalves; ++t) {
                v_bad = v_bad || (any[t] && vs[t] != vs[t]);
                const float lift = any[t] ? scale_log(vs[t], v_exp) : 0.0f, base = (float)kBias - top + lift;
                float run = 0.0f, w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][e], factor[t], base));
                    run += w[e];
                }
                sum = __builtin_fmaf(run, __builtin_amdgcn_exp2f(-lift), sum);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h2 u, v;
                    split_pair(w[2 * e], w[2 * e + 1], &u, &v);
                    wh[2 * t + e / 4][2 * e % 8] = u[0], wh[2 * t + e / 4][2 * e % 8 + 1] = u[1];
                    wl[2 * t + e / 4][2 * e % 8] = v[0], wl[2 * t + e / 4][2 * e % 8 + 1] = v[1];
                }
            }
#pragma unroll
            for (int k = 0; k < kOut; ++k)
#pragma unroll
                for (int t = 0; t < 2 * kHalves; ++t) {  // tokens 32 (half0 + t / 2) + 16 hf + 8 (t % 2) ..
                    const h8 val = *reinterpret_cast<const h8*>(&st.v[k * 32 + col][(half0 + t / 2) * 32 + hf * 16 + (t % 2) * 8]);
                    o[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(val, wh[t], o[k], 0, 0, 0);
                    o[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(val, wl[t], o[k], 0, 0, 0);
                }
        }
        if (more) store(stage[(p + 1 - p0) & 1]);
        __syncthreads();
    }
    bad = __syncthreads_or(bad) != 0;
    if constexpr (KS == 2) {  // the second halves' results join the first's, register by register, through the pages' LDS
        float* mine = reinterpret_cast<float*>(smem) + wave / 2 * (kOut * 16 + 4) * 64 + lane;
        if (half0 == 1) {
#pragma unroll
            for (int k = 0; k < kOut; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) mine[(k * 16 + e) * 64] = o[k][e];
            mine[kOut * 16 * 64] = top;
            mine[(kOut * 16 + 1) * 64] = sum;
            mine[(kOut * 16 + 2) * 64] = v_exp;
            mine[(kOut * 16 + 3) * 64] = v_bad ? 1.0f : 0.0f;
        }
        __syncthreads();
        if (half0 == 1) return;
        const float top2 = mine[kOut * 16 * 64], new_top = fmaxf(top, top2);
        const float e1 = v_exp + (top - new_top), e2 = mine[(kOut * 16 + 2) * 64] + (top2 - new_top), new_exp = fmaxf(fmaxf(e1, e2), kNoExp);
        const float f1 = __builtin_amdgcn_exp2f(top - new_top), f2 = __builtin_amdgcn_exp2f(top2 - new_top);
        const float o1 = __builtin_amdgcn_exp2f(e1 - new_exp), o2 = __builtin_amdgcn_exp2f(e2 - new_exp);
#pragma unroll
        for (int k = 0; k < kOut; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[k][e] = __builtin_fmaf(mine[(k * 16 + e) * 64], o2, o[k][e] * o1);
        sum = __builtin_fmaf(mine[(kOut * 16 + 1) * 64], f2, sum * f1);
        v_bad = v_bad || mine[(kOut * 16 + 3) * 64] != 0.0f;
        top = new_top;
        v_exp = new_exp;
    }
    sum = halves_sum(sum);
    if (halves_max(v_bad ? 1.0f : 0.0f) > 0.0f)
#pragma unroll
        for (int k = 0; k < kOut; ++k) o[k] = (f16x)(__builtin_nanf(""));
    if (!live) return;
    // (the unit comes last: before it the numbers are of ordinary size, whatever the values are)
    const float nan = __builtin_nanf(""), up = __builtin_amdgcn_exp2f(v_exp), scale = bad ? nan : sum == 0.0f ? 0.0f : 1.0f / sum;
    if (parts > 1) {
        float* piece = scratch + ((((size_t)s * c.n_kv + h) * tiles + rt) * parts + part) * kPieceFloats<DP, KS>;
        const int r = wave / KS * kCols + col;
#pragma unroll
        for (int k = 0; k < kOut; ++k)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<f4*>(&piece[r * DP + k * 32 + 2 * e + 4 * hf]) = f4{o[k][e], o[k][e + 1], o[k][e + 2], o[k][e + 3]} * scale * up;
        if (hf == 0) {
            piece[kRows * DP + r] = top;
            piece[kRows * DP + kRows + r] = bad ? nan : sum * pow2(-kSumDown);
        }
        return;
    }
    const size_t at = (size_t)(q.r0 + i) * a.n_head + head;
    float* out = dst + at * c.dim;
    const bool vec = c.dim % 4 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
#pragma unroll
    for (int k = 0; k < kOut; ++k)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = k * 32 + 2 * e + 4 * hf;
            const f4 y = f4{o[k][e], o[k][e + 1], o[k][e + 2], o[k][e + 3]} * scale * up;
            if (vec) {
                if (d < c.dim) *reinterpret_cast<f4*>(out + d) = y;
            } else {
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (d + n < c.dim) out[d + n] = y[n];
            }
        }
    if (lse && hf == 0)
        lse[at] = bad ? nan : sum == 0.0f ? -__builtin_inff() : (__builtin_amdgcn_logf(sum) + top - (float)kBias) * kLn2;
}

// Joins the pieces of the rows of one (sequence, head, row tile), a wave at a time per row.
template <int DP, int KS>
__global__ __launch_bounds__(kThreads) void join_rows_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a, float* __restrict__ dst,
                                                             float* __restrict__ lse, const float* __restrict__ scratch,
                                                             int tiles, int parts) {
    constexpr int kRows = infr::kRows<KS>;
    const int lane = threadIdx.x & 63;
    const int rt = blockIdx.x % tiles, h = blockIdx.x / tiles % c.n_kv, s = blockIdx.x / tiles / c.n_kv;
    const int r = (int)blockIdx.y * kWaves + ((int)threadIdx.x >> 6), r_all = rt * kRows + r;
    const Kv8Seq q = kv8_seq(b, s);
    if (r_all >= q.n * a.group) return;
    const float* first = scratch + (((size_t)s * c.n_kv + h) * tiles + rt) * parts * kPieceFloats<DP, KS>;
    float m = kNoMax, l = 0.0f;
    for (int k = 0; k < parts; ++k) m = fmaxf(m, first[(size_t)k * kPieceFloats<DP, KS> + kRows * DP + r]);
    float x[DP / 64] = {};  // (columns behind head_dim are whatever the scratch held; they are not stored)
    for (int k = 0; k < parts; ++k) {
        const float* piece = first + (size_t)k * kPieceFloats<DP, KS>;
        const float f = piece[kRows * DP + kRows + r] * __builtin_amdgcn_exp2f(piece[kRows * DP + r] - m);
        l += f;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) x[j] += piece[r * DP + j * 64 + lane] * f;
    }
    const size_t at = (size_t)(q.r0 + r_all / a.group) * a.n_head + h * a.group + r_all % a.group;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j)
        if (j * 64 + lane < c.dim) dst[at * c.dim + j * 64 + lane] = l == 0.0f ? 0.0f : l != l ? l : x[j] / l;
    if (lse && lane == 0) lse[at] = l == 0.0f ? -__builtin_inff() : (__builtin_amdgcn_logf(l) + m - (float)(kBias - kSumDown)) * kLn2;
}

int tiles_of(int group, int max_q, int ks) {
    const int rows = kCols * kWaves / ks;
    return (int)(((int64_t)max_q * group + rows - 1) / rows);
}

// How a call is cut up.
struct Cut {
    int ks, tiles, parts;
};
// Row tiles for waves that share rows by ks, and the parts their pages are cut into: enough for two workgroups on each
// compute unit, of at least eight pages where sequences are as long as the page table is wide.
Cut cut_for(int ks, int cus, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    Cut c;
    c.ks = ks;
    c.tiles = tiles_of(group, max_q, ks);
    const int64_t wgs = (int64_t)n_seq * n_kv * c.tiles;
    c.parts = (int)std::max<int64_t>(1, std::min<int64_t>(2 * cus / wgs, max_pages / 8));
    return c;
}
// Two waves to 32 rows halve a workgroup's time per page and double what is spent on bringing pages into LDS: better while
// the time is that of the longest row tiles, which is up to four tiles of 128 rows for a compute unit (one / two ways, 32
// heads of 128, 8 KV heads, short bursts: 512 tokens 30 / 22 us, 1024 51 / 40, 2048 104 / 99, four times 1024 109 / 125, 4096 300 / 328;
// three packed prompts, 16 heads of 80: 88 / 67), two with more than 128 columns, where a compute unit holds one workgroup
// (256 columns: 1024 tokens 96 / 80, 2048 197 / 252). Not where the twice as many tiles leave less than half the parts
// (300 rows each behind 3000 and 1500 tokens, three parts / one: 82 / 98).
Cut cut_of(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    const Cut one = cut_for(1, cus, n_kv, group, n_seq, max_q, max_pages), two = cut_for(2, cus, n_kv, group, n_seq, max_q, max_pages);
    const bool few = (int64_t)n_seq * n_kv * one.tiles < (int64_t)(dim <= 128 ? 4 : 2) * cus;
    return few && 2 * two.parts >= one.parts ? two : one;
}

template <int DP, int DC, int KS>
void launch_prompt_ks(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch, const Cut& cut,
                      hipStream_t stream) {
    const bool gen = a.softcap > 0.0f || a.window > 0 || a.slopes || a.first || a.prefix;
    auto kernel = c.f8 ? (gen ? prompt_kernel<DP, DC, KS, true, true> : prompt_kernel<DP, DC, KS, true, false>)
                       : (gen ? prompt_kernel<DP, DC, KS, false, true> : prompt_kernel<DP, DC, KS, false, false>);
    const size_t lds = 2 * sizeof(Stage<DC>);
    static_assert(2 * sizeof(Stage<DC>) >= kWaves / 2 * (DC / 2 + 4) * 64 * sizeof(float), "the second halves' results fit");
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    // heads side by side: workgroups go round the XCDs in this order, so a head's pages stay in one L2
    hipLaunchKernelGGL(kernel, dim3((unsigned)(c.n_kv * cut.parts), (unsigned)b.n_seq, (unsigned)cut.tiles), dim3(kThreads), lds,
                       stream, c, b, a, dst, lse, scratch, cut.tiles, cut.parts);
    if (cut.parts > 1)
        hipLaunchKernelGGL((join_rows_kernel<DP, KS>), dim3((unsigned)(b.n_seq * c.n_kv * cut.tiles), kRows<KS> / kWaves),
                           dim3(kThreads), 0, stream, c, b, a, dst, lse, scratch, cut.tiles, cut.parts);
}
template <int DP, int DC>
void launch_prompt_dc(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch, int cus,
                      hipStream_t stream) {
    const Cut cut = cut_of(cus, c.dim, c.n_kv, a.group, b.n_seq, b.max_q, b.max_pages);
    if (cut.ks == 2) launch_prompt_ks<DP, DC, 2>(c, b, a, dst, lse, scratch, cut, stream);
    else launch_prompt_ks<DP, DC, 1>(c, b, a, dst, lse, scratch, cut, stream);
}
template <int DP>
void launch_prompt_dp(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch, int cus,
                      hipStream_t stream) {
    if (c.dim <= DP - 32) launch_prompt_dc<DP, DP - 32>(c, b, a, dst, lse, scratch, cus, stream);
    else launch_prompt_dc<DP, DP>(c, b, a, dst, lse, scratch, cus, stream);
}

}  // namespace

size_t prompt_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    const Cut cut = cut_of(cus, dim, n_kv, group, n_seq, max_q, max_pages);
    const size_t dp = (size_t)(dim + 63) / 64 * 64, rows = kCols * kWaves / cut.ks;
    return cut.parts == 1 ? 0 : (size_t)n_seq * n_kv * cut.tiles * cut.parts * (rows * dp + 2 * rows) * sizeof(float);
}
void launch_attention_prompt(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch,
                             int cus, hipStream_t stream) {
    switch (c.dp) {
    case 64: launch_prompt_dp<64>(c, b, a, dst, lse, scratch, cus, stream); break;
    case 128: launch_prompt_dp<128>(c, b, a, dst, lse, scratch, cus, stream); break;
    case 192: launch_prompt_dp<192>(c, b, a, dst, lse, scratch, cus, stream); break;
    default: launch_prompt_dp<256>(c, b, a, dst, lse, scratch, cus, stream); break;
    }
}

}  // namespace infr
