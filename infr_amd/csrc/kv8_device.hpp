// Device pieces that the kernels reading the 8-bit KV cache share: codes to f16, f32 operands as two f16
// numbers, the scores' softcap, bias and masks.
//
// Matrix products run on the f16 MFMA. Every code of either type is exact in f16; an f32 operand x goes in as
// hi + lo, hi = f16(x) and lo = f16(x - hi), two products instead of one, so that 23 bits of it count (f16 alone
// would leave 11, which shows in an f32 result). Query rows are scaled by a power of two that puts their largest
// value at 2^14, softmax weights by 2^11, so that the smallest f16 number stands far below what counts.
//
// Layouts follow from S^T = K Q^T: with tokens as the MFMA's rows and query rows as its columns, a lane's scores
// all belong to one query row, the softmax statistics of a row live in the lanes that hold its output, and the
// weights are P.V's operand where they stand: no exchange between lanes but the maximum's.
#pragma once

#include "kv8.hpp"

namespace infr {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16x __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoMax = -3.4028234e38f;  // running maximum before the first token: finite, so that -inf - it is -inf

// 16 bytes of codes that are read once and, with their neighbours in the wave, in whole lines: non-temporal (a decode
// step over 360 MB of cache measured 80 us so against 89 us with plain loads).
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const u4 x = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// Exponents are formed as fma(product, factor, -maximum), with the maximum rounded and the product not: they miss by
// half an ulp of the score, the same for all of a row. Above this size, where that could be more than 2^-8, the scores
// are rounded first.
constexpr float kLargeScore = 65536.0f;

// Two codes (bytes 2 * word, 2 * word + 1 of c) as f16.
template <bool F8>
__device__ __forceinline__ h2 code_pair(uint32_t c, int word) {
    if constexpr (F8) {
        return word ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false);
    } else {
        // 0x6400 | u is 1024 + u; with u = code + 128 the difference to 1152 is the code, exactly
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, c ^ 0x80808080u, word ? 0x04030402u : 0x04010400u);
        return __builtin_bit_cast(h2, u) - (h2)(_Float16)1152.0f;
    }
}
template <bool F8>
__device__ __forceinline__ h8 code_oct(uint32_t a, uint32_t b) {
    const h2 p = code_pair<F8>(a, 0), q = code_pair<F8>(a, 1), r = code_pair<F8>(b, 0), s = code_pair<F8>(b, 1);
    return h8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// a, b = hi + lo, both rounded to the nearest (one instruction for two numbers): 23 bits of each remain, and what falls off
// falls to either side.
__device__ __forceinline__ h2 nearest_pair(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector(f2{a, b}, h2);
}
__device__ __forceinline__ void split_pair(float a, float b, h2* hi, h2* lo) {
    *hi = nearest_pair(a, b);
    *lo = nearest_pair(__builtin_fmaf((float)(*hi)[0], -1.0f, a), __builtin_fmaf((float)(*hi)[1], -1.0f, b));
}

// f over lanes l and l ^ 32.
template <typename F>
__device__ __forceinline__ float across_halves(float x, F f) {
    // (the elements are copied before they are reinterpreted: a bit cast of a vector's element reads its first one)
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float halves_max(float x) {
    return across_halves(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float halves_sum(float x) {
    return across_halves(x, [](float a, float b) { return a + b; });
}
// Maximum / sum over lanes l, l ^ 16, l ^ 32, l ^ 48.
template <typename F>
__device__ __forceinline__ float across_quads(float x, F f) {
    const uint32_t w = __builtin_bit_cast(uint32_t, across_halves(x, f));
    const auto q = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    const uint32_t c = q[0], d = q[1];
    return f(__builtin_bit_cast(float, c), __builtin_bit_cast(float, d));
}
__device__ __forceinline__ float quads_max(float x) {
    return across_quads(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float quads_sum(float x) {
    return across_quads(x, [](float a, float b) { return a + b; });
}

// Power of two that brings a query row with this largest |value| to 2^14; rows of zeros and of values too small
// or too large for it get the nearest that keeps every factor a normal number.
__device__ __forceinline__ int row_exponent(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 14;
    return min(max(e, -100), 114);
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

// N floats of a row of `dim` from column d0 on, zeros behind its end; N is a multiple of 4 and so is d0. `vec`: the
// row's length is a multiple of 4 and it is aligned to 16 bytes.
template <int N>
__device__ __forceinline__ void load_row(const float* x, int d0, int dim, bool live, bool vec, float* v) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const int d = d0 + e;
        f4 y = f4{0, 0, 0, 0};
        if (live && d < dim) {
            if (vec) y = *reinterpret_cast<const f4*>(x + d);
            else
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = d + k < dim ? x[d + k] : 0.0f;
        }
        v[e] = y[0], v[e + 1] = y[1], v[e + 2] = y[2], v[e + 3] = y[3];
    }
}
__device__ __forceinline__ bool rows_vec(const Kv8Cache& c, const Kv8Attn& a) {
    return c.dim % 4 == 0 && a.q_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
}

// 1 / c, finite for every c > 0: a score of 0 is capped to 0, whatever c is.
__device__ __forceinline__ float inverse_cap(float c) { return c > 0.0f ? fminf(1.0f / c, 3.4028234e38f) : 0.0f; }

// x[i] = c * tanh(x[i] / c), to the last bits of x (with x and c both times log2 e it is the capped score times that).
// Scores are mostly small beside the cap: where all of a wave's are below a quarter of it, four terms of tanh's series
// serve (the fifth is under 2^-26). Else six below 0.35, and 1 - 2 / (e^2y + 1) beyond, whose difference cancels no more
// than two bits.
// FOURS: four of them at a time, where all at once would spill. inv_c: inverse_cap(c).
template <int N, bool FOURS, typename X>
__device__ __forceinline__ void cap_scores(X& x, float c, float inv_c) {
    float most = fabsf(x[0]);
#pragma unroll
    for (int e = 1; e < N; ++e) most = fmaxf(most, fabsf(x[e]));
    if (__all(most * inv_c < 0.25f)) {  // (a NaN among others does not show in `most`; the series passes it on)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float y = x[e] * inv_c, z = y * y;
            float p = __builtin_fmaf(62.0f / 2835.0f, z, -17.0f / 315.0f);
            p = __builtin_fmaf(p, z, 2.0f / 15.0f);
            p = __builtin_fmaf(p, z, -1.0f / 3.0f);
            x[e] = __builtin_fmaf(x[e], p * z, x[e]);
            if (FOURS && e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float s = x[e], y = fabsf(s) * inv_c, z = y * y;
            float p = __builtin_fmaf(-1382.0f / 155925.0f, z, 62.0f / 2835.0f);
            p = __builtin_fmaf(p, z, -17.0f / 315.0f);
            p = __builtin_fmaf(p, z, 2.0f / 15.0f);
            p = __builtin_fmaf(p, z, -1.0f / 3.0f);
            const float near = __builtin_fmaf(s, p * z, s), d = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e)) + 1.0f;
            float r = __builtin_amdgcn_rcpf(d);
            r = __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.0f), r);
            const float far = __builtin_copysignf(c * (1.0f - 2.0f * (d < __builtin_inff() ? r : 0.0f)), s);
            x[e] = y >= 0.35f ? far : near;
            if (FOURS && e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Softmax weights go into P.V times the scale of their value's block and 2^(kBias - v_exp). v_exp follows the largest product
// of weight and scale, so that what carries the row keeps its bits however far its scale is below that of a block of next
// to no weight (with v_exp by the scales alone, a block 2^24 below such a one lost 8e-5 of its sum, at 2^36 all of it).
// Weights count from the running maximum `top`, and so does v_exp; both may lag behind by 2^kLag, which keeps the
// products below 2^15 (f16 ends at 2^16). The largest one stands at 2^9 or above: what is 2^-34 of it is below f16's
// smallest numbers and rounded away.
constexpr int kBias = 11;
constexpr float kLag = 4.0f;
constexpr float kNoExp = -400.0f;  // v_exp before the first token: below any product's exponent
// A piece of a row's keys leaves its own softmax's output, no larger than the values are, with its maximum and its sum of
// weights; the latter by 2^-kSumDown, which is below 1 for 2^22 tokens, so that outputs times sums are no larger either.
constexpr int kSumDown = 40;

// Exponent that the product of a block's scale and its largest weight stays below; -inf for a NaN scale and where no
// token is seen (`high` is -inf then).
__device__ __forceinline__ float product_exponent(float scale, float high, float top) {
    const int e = (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255u) - 126;
    return scale < __builtin_inff() ? (float)e + (high - top) : -__builtin_inff();
}
// A block's value scale as the weights' exponent: log2 of scale / 2^v_exp. Weights of 2^-60 and less are 0 in f16, and from
// there on the exponent stays as it is, so that their sum, which is divided by it again, keeps clear of the smallest numbers.
__device__ __forceinline__ float scale_log(float scale, float v_exp) {
    const float l = __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(scale)) + ((float)__builtin_amdgcn_frexp_expf(scale) - v_exp);
    return scale < __builtin_inff() ? fmaxf(l, -60.0f) : 0.0f;  // a NaN scale is the caller's
}

// What one query row sees, and its bias.
struct Kv8Row {
    int slot, pos, first, prefix, window;  // slot: last token by causality; prefix: positions below it are seen always
    float slope;                           // times log2 e; 0: none
    __device__ __forceinline__ bool sees(int token, int kpos) const {
        return (token <= slot || kpos < prefix) && pos - kpos < window && kpos >= first;
    }
};
// Row i of sequence s, head `head`. Positions are taken to lie in [0, 2^30].
__device__ __forceinline__ Kv8Row kv8_row(const Kv8Batch& b, const Kv8Attn& a, const Kv8Seq& q, int s, int i, int head) {
    Kv8Row r;
    r.slot = a.causal ? q.len - q.n + i : 0x7FFFFFFF;
    r.pos = b.pos[q.r0 + i];
    r.first = a.first ? a.first[q.r0 + i] : -0x7FFFFFFF - 1;
    r.prefix = a.prefix ? a.prefix[s] : -0x7FFFFFFF - 1;
    r.window = a.window > 0 ? a.window : 0x7FFFFFFF;
    r.slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    return r;
}

// ---- how the kernels for few rows cut a batch's pages: pieces of one size, found from the lengths ----

constexpr int kStepWaves = 4;   // waves of a workgroup, each a page at a time
constexpr int kStepRows = 16;   // query rows of a workgroup, or half of them: see step_rows

// Row tiles, first page any row sees, pages from there. `all`: every cached page is gone over by one tile, whether
// rows see it or not (ScoreKv8 lets sums decay).
struct SeqWork {
    int tiles, p_lo, pages;
};
__device__ __forceinline__ SeqWork seq_work(const Kv8Seq& q, const Kv8Attn& a, int rows, bool all) {
    SeqWork w;
    w.tiles = all ? 1 : (q.n * a.group + rows - 1) / rows;
    w.p_lo = 0;
    w.pages = 1;  // of a sequence whose tables are wrong one item per tile writes the rows' NaN
    if (q.ok) {
        // positions ascend with the tokens, so a token `window` or more tokens back is outside the window
        const int lo = a.window > 0 && !all ? max(q.len - q.n - a.window + 1, 0) : 0;
        w.p_lo = lo / kPage;
        w.pages = max((q.len + kPage - 1) / kPage - w.p_lo, 1);
    }
    return w;
}

// Value of lane l ^ 8 (within rows of 16 lanes, which a rotation by 8 swaps the halves of).
__device__ __forceinline__ float from_other_eight(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xF, 0xF, true));
}

// The query rows of a workgroup in LDS as f16, scaled by their powers of two (factor: what a product of codes is to be
// multiplied by, times log2 e): low parts behind the high ones (with
// ROWS = 8 the two are the 16 columns of one MFMA). Rows are padded by 16 bytes.
template <int DP, int ROWS>
struct StepQ {
    _Float16 x[2 * ROWS][DP + 8];
    float factor[ROWS];
};
// 256 threads bring in rows 0 .. ROWS - 1 of `tile`, row by row side by side.
template <int DP, int ROWS>
__device__ __forceinline__ void stage_rows(StepQ<DP, ROWS>& st, const Kv8Cache& c, const Kv8Attn& a, const Kv8Seq& q, int h, int row0) {
    constexpr int kEach = ROWS, kSide = 256 / ROWS;  // threads of a row; each four columns at a time
    constexpr int kFours = (DP / 4 + kSide - 1) / kSide;
    static_assert(kEach * kSide == 256, "a workgroup of 256");
    const int r = (int)threadIdx.x / kSide, t = (int)threadIdx.x % kSide, rr = row0 + r;
    const bool live = rr < q.n * a.group, vec = rows_vec(c, a);
    const float* x = a.q;
    if (live) x += (size_t)(q.r0 + rr / a.group) * a.q_stride + (size_t)(h * a.group + rr % a.group) * c.dim;
    float v[4 * kFours];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kFours; ++k) {
        load_row<4>(x, (k * kSide + t) * 4, c.dim, live, vec, v + 4 * k);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, abs_bits(v[4 * k + e]));
    }
#pragma unroll
    for (int o = 1; o < kSide; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    const int e2 = row_exponent(top);
    const float down = a.scale < 0.0f ? -pow2(-e2) : pow2(-e2);  // factors stay positive: a maximum may be taken before them
#pragma unroll
    for (int k = 0; k < kFours; ++k) {
        const int d = (k * kSide + t) * 4;
        h2 h0, h1, l0, l1;
        split_pair(v[4 * k] * down, v[4 * k + 1] * down, &h0, &l0);
        split_pair(v[4 * k + 2] * down, v[4 * k + 3] * down, &h1, &l1);
        if (d < DP) {
            *reinterpret_cast<h4*>(&st.x[r][d]) = h4{h0[0], h0[1], h1[0], h1[1]};
            *reinterpret_cast<h4*>(&st.x[ROWS + r][d]) = h4{l0[0], l0[1], l1[0], l1[1]};
        }
    }
    if (t == 0) st.factor[r] = fabsf(a.scale) * kLog2e * pow2(e2);
}

// A sequence's share of the pieces: `parts` of each (head, row tile), the first of them number `first`.
struct SeqCut {
    int s;  // -1: none
    Kv8Seq q;
    SeqWork work;
    int parts, first;
};
// The share of sequence `want`, or, with want < 0, of the sequence that holds piece `item`. About `target` pieces are
// aimed at, of at least one page for each wave of a workgroup; sequences of up to `whole` pages are one. Up to 64
// sequences take one round of loads, and the sequence found is passed between the lanes; more of them take a loop over the
// tables and another over the counts.
__device__ __forceinline__ SeqCut find_cut(const Kv8Batch& b, const Kv8Attn& a, int n_kv, int rows, int target, int whole, bool all,
                                           int want, int item) {
    const int lane = (int)(threadIdx.x & 63);
    Kv8Seq q{};
    SeqWork w{};
    float total = 0.0f;
    for (int s = lane; s < b.n_seq; s += 64) {
        q = kv8_seq(b, s);
        w = seq_work(q, a, rows, all);
        total += (float)w.tiles * (float)w.pages;
    }
    total = wave_total(total);
    const int size = max((int)__builtin_ceilf(total * (float)n_kv / (float)target), kStepWaves);
    SeqCut r;
    r.s = -1;
    int before = 0;
    for (int base = 0; base < b.n_seq; base += 64) {
        const int s = base + lane;
        if (b.n_seq > 64) {
            if (s < b.n_seq) {
                q = kv8_seq(b, s);
                w = seq_work(q, a, rows, all);
            }
        }
        const int parts = s < b.n_seq ? (w.pages <= whole ? 1 : (w.pages + size - 1) / size) : 0, n = n_kv * w.tiles * parts;
        const int sum = wave_scan(s < b.n_seq ? n : 0);
        const unsigned long long hit = __ballot(want >= 0 ? s == want : item - before < sum);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            r.s = base + l;
            r.q.r0 = of(q.r0);
            r.q.n = of(q.n);
            r.q.len = of(q.len);
            r.q.ok = of((int)q.ok) != 0;
            r.work.tiles = of(w.tiles);
            r.work.p_lo = of(w.p_lo);
            r.work.pages = of(w.pages);
            r.parts = of(parts);
            r.first = before + of(sum) - of(n);
            return r;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return r;
}

}  // namespace infr
