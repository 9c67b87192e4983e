// AttentionKv8 for few rows per sequence: decode steps and drafts. Bound by reading the cache once.
//
// Up to 16 query rows of one (sequence, KV head) - its rows times the heads of the group - are one column tile of
// the 16x16x32 f16 MFMA; up to 8 of them take its other 8 columns for their low parts, and half the products. A wave
// takes one page at a time: 64 tokens as four row tiles chosen so that lane group g holds tokens 16 g .. 16 g + 15 of
// its query row, which is what P.V wants side by side from V^T's 16-byte pieces. Key and value codes go from HBM to
// registers in 16-byte loads (whole lines per instruction), become f16 there and feed the MFMA; the next page's keys
// are requested before the current page's softmax, its values before its scores.
//
// The pages of all sequences are cut into pieces of one size, found on the device from the lengths: long sequences
// get many workgroups, short ones one, and no piece is empty. A sequence in one piece writes its result; the pieces
// of others are joined by a second kernel, in their order.
// Measured (8 KV heads of 128, 32 heads): one token of 64 sequences of 500 to 8000 tokens 71 us, 5.1 TB/s, 63 us and 5.7
// TB/s of it the first kernel (a pass that only reads: 7.1 TB/s); two sequences of 115000 tokens, 4 KV heads, 46 us, 5.2
// TB/s; one of 700 tokens 10.3 us, launch and dependent loads; drafts of 4 tokens of 16 sequences, window 1024, capped, 8
// KV heads of 256, 22 us, bound by what one wave does for half a page. (A join by the workgroup that comes last to its row tile
// saves that launch but costs its own round trips past the L2, which the XCDs do not share: 53 us against 49 for two
// sequences of 115000 tokens, 48 against 44 for drafts of four tokens.)
#include <type_traits>

#include "kv8_attn.hpp"
#include "kv8_device.hpp"

namespace infr {

namespace {

// Waves of a workgroup that take TOK tokens of a page at a time: together four pages.
template <int TOK>
constexpr int kWaves = kPage / TOK * kStepWaves;

// Outputs, maxima and sums of a piece: f32 [rows][DP], then [rows] pairs of a maximum and a sum.
template <int DP, int ROWS>
constexpr int kPieceFloats = ROWS * DP + 2 * ROWS;

template <int DP, int ROWS, int TOK, bool F8, bool GEN>
__global__ __launch_bounds__(64 * kWaves<TOK>, DP == 64 ? 3 : DP == 128 || (DP == 192 && ROWS == 8) || TOK == 32 ? 2 : 1) void step_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a,
                                                                             float* __restrict__ dst, float* __restrict__ lse,
                                                                             float* __restrict__ scratch, int target, int whole_pages) {
    constexpr int kCols = DP / 64;   // 64-column groups of a key
    constexpr int kOut = DP / 16;    // 16-column groups of a value
    constexpr int kWaves = infr::kWaves<TOK>, kFours = DP / 4, kThreads = 64 * kWaves;
    constexpr int kShare = kPage / TOK;                  // waves that share a page
    constexpr int kMine = TOK / 4, kTiles = TOK / 16;    // tokens of a lane; row tiles of the MFMA
    constexpr int kPart = ROWS * (DP + 4);
    constexpr bool PACK = ROWS == 8;   // columns 8..15 are the low parts of columns 0..7
    __shared__ __align__(16) float part_o[kWaves * kPart];  // the waves' outputs; before, the query rows
    static_assert(sizeof(StepQ<DP, ROWS>) <= sizeof(part_o), "the rows fit");
    __shared__ float part_m[kWaves][16], part_l[kWaves][16], part_e[kWaves][16], row_e[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const SeqCut cut = find_cut(b, a, c.n_kv, ROWS, target, whole_pages, false, -1, (int)blockIdx.x);
    if (cut.s < 0) return;
    const int s = cut.s, parts = cut.parts, rest = (int)blockIdx.x - cut.first;
    const Kv8Seq q = cut.q;
    const SeqWork work = cut.work;
    const int part = rest % parts, rt = rest / parts % work.tiles, h = rest / parts / work.tiles;
    const int per = (work.pages + parts - 1) / parts;
    const int p0 = work.p_lo + part * per;
    const int p1 = q.ok ? min(p0 + per, (q.len + kPage - 1) / kPage) : p0;
    const int n_rows = q.n * a.group;
    const int rr = rt * ROWS + col % ROWS;                   // this lane's query row
    const bool live = rr < n_rows;
    const int i = live ? rr / a.group : q.n - 1, head = h * a.group + (live ? rr % a.group : 0);

    const Kv8Row row = kv8_row(b, a, q, s, i, head);
    const float cap = a.softcap * kLog2e, inv_cap = GEN ? inverse_cap(cap) : 0.0f;
    const bool use_pos = GEN && (a.window > 0 || a.slopes || a.first || a.prefix);
    // tokens below this one are seen by every row of the tile (without masks by position)
    const int all_see = a.causal ? q.len - q.n + rt * ROWS / a.group + 1 : q.len;

    int last_pos = live ? row.pos : -0x7FFFFFFF - 1, last_first = live ? row.first : -0x7FFFFFFF - 1;
    if (use_pos)
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) {
            last_pos = max(last_pos, __shfl_xor(last_pos, k));
            last_first = max(last_first, __shfl_xor(last_first, k));
        }

    f4 o[kOut];
#pragma unroll
    for (int k = 0; k < kOut; ++k) o[k] = f4{0, 0, 0, 0};
    float top = kNoMax, sum = 0.0f;
    float v_exp = kNoExp;  // O's unit: 2^v_exp / 2^kBias
    bool bad = !q.ok, v_bad = false;  // v_bad: the row sees a token whose value is NaN

    const int32_t* table = b.pages + (size_t)s * b.max_pages;
    const int subs = kPage / c.block;
    const uint32_t kv_stride = (uint32_t)DP * kPage;
    using VCodes = typename std::conditional<TOK == 64, uint4, uint2>::type;
    uint4 kf[kTiles][kCols];
    VCodes vf[kOut];
    float ks = 0.0f, vs = 0.0f;
    int page = 0, ids = 0, pos0 = 0;
    const int half = wave % kShare * TOK;  // the wave's first token in a page
    // lane n holds the wave's n-th next page
    auto load_ids = [&](int p) {
        const int at = p + lane * kStepWaves;
        ids = at < p1 ? table[at] : 0;
        if (ids < 0 || ids >= c.n_pages) ids = -1;
        if (__any(ids < 0)) bad = true;
    };
    auto load_keys = [&](int n) {
        page = max(__builtin_amdgcn_readlane(ids, n), 0);
        const uint8_t* kp = c.k + ((size_t)page * c.n_kv + h) * kv_stride + (half + kMine * (col >> 2) + (col & 3)) * 64 + 16 * g;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int j = 0; j < kCols; ++j) kf[t][j] = load_stream(kp + j * kPage * 64 + t * 4 * 64);
        const size_t sc = ((size_t)page * c.n_kv + h) * subs + (half + g * kMine) / c.block;
        ks = c.ks[sc];
        vs = c.vs[sc];
        if (use_pos) pos0 = c.pos[((size_t)page * c.n_kv + h) * kPage];
    };
    int p = p0 + wave / kShare, n = 0;
    if (p < p1) {
        load_ids(p);
        load_keys(0);
    }
    // the query rows as hi + lo
    StepQ<DP, ROWS>& rows_q = *reinterpret_cast<StepQ<DP, ROWS>*>(part_o);
    if (kWaves == 4 || wave < 4) stage_rows<DP, ROWS>(rows_q, c, a, q, h, rt * ROWS);  // (whole waves, 256 threads)
    __syncthreads();
    h8 qh[2 * kCols], ql[PACK ? 1 : 2 * kCols];
#pragma unroll
    for (int k = 0; k < 2 * kCols; ++k) {
        const int d = (k / 2) * 64 + g * 16 + (k % 2) * 8;
        qh[k] = *reinterpret_cast<const h8*>(&rows_q.x[col][d]);
        if constexpr (!PACK) ql[k] = *reinterpret_cast<const h8*>(&rows_q.x[16 + col][d]);
    }
    const float row_factor = rows_q.factor[col % ROWS];
    while (p < p1) {
        const uint8_t* vp = c.v + ((size_t)page * c.n_kv + h) * kv_stride + col * kPage + half + kMine * g;
#pragma unroll
        for (int k = 0; k < kOut; ++k) {
            if constexpr (TOK == 64) vf[k] = load_stream(vp + k * 16 * kPage);
            else vf[k] = *reinterpret_cast<const uint2*>(vp + k * 16 * kPage);  // (the other half of the line is another wave's)
        }
        // (positions ascend: what the tile's last row's window and document allow at the page's first token, all rows do)
        const bool masked = (p + 1) * kPage > min(all_see, q.len) || (use_pos && (last_pos - pos0 >= row.window || last_first > pos0));
        int kpos[kMine];
        if (use_pos && (masked || a.slopes)) {
            const int4* pp = reinterpret_cast<const int4*>(c.pos + ((size_t)page * c.n_kv + h) * kPage + half + kMine * g);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int4 x = pp[t];
                kpos[4 * t] = x.x, kpos[4 * t + 1] = x.y, kpos[4 * t + 2] = x.z, kpos[4 * t + 3] = x.w;
            }
        }
        // scores: sc[t][i] is token kMine g + 4 t + i of the wave's
        f4 sc[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            sc[t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                const h8 lo = code_oct<F8>(kf[t][j].x, kf[t][j].y), hi = code_oct<F8>(kf[t][j].z, kf[t][j].w);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qh[2 * j], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qh[2 * j + 1], sc[t], 0, 0, 0);
                if constexpr (!PACK) {
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, ql[2 * j], sc[t], 0, 0, 0);
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ql[2 * j + 1], sc[t], 0, 0, 0);
                }
            }
        }
        const int tok0 = p * kPage + half + kMine * g;
        const float factor = row_factor * ks;
        const float vs_now = vs;
        const bool tail = (p + 1) * kPage > q.len;
        // the next page's keys are on their way from here
        const int np = p + kStepWaves;
        if (np < p1) {
            if (++n == 64) {
                load_ids(np);
                n = 0;
            }
            load_keys(n);
        }
        float x[kMine], f = factor;
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            float v = sc[e / 4][e % 4];
            if (PACK) v += from_other_eight(v);
            x[e] = v;
        }
        if (masked || (GEN && (a.softcap > 0.0f || a.slopes))) {
#pragma unroll
            for (int e = 0; e < kMine; ++e) x[e] *= factor;
            if (GEN && a.softcap > 0.0f) cap_scores<kMine, false>(x, cap, inv_cap);
            if (GEN && a.slopes)
#pragma unroll
                for (int e = 0; e < kMine; ++e) x[e] = __builtin_fmaf(-row.slope, fabsf((float)(row.pos - kpos[e])), x[e]);
            f = 1.0f;
        }
        bool any = true;
        if (masked) {
            any = false;
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                const int tok = tok0 + e;
                const bool yes = tok < q.len && (use_pos ? row.sees(tok, kpos[e]) : tok <= row.slot);
                any = any || yes;
                x[e] = yes ? x[e] : -__builtin_inff();
            }
        }
        float high = x[0];
#pragma unroll
        for (int e = 1; e < kMine; ++e) high = fmaxf(high, x[e]);
        high *= f;
        if (__any(fabsf(high) > kLargeScore)) {
#pragma unroll
            for (int e = 0; e < kMine; ++e) x[e] *= f;
            f = 1.0f;
        }
        if (__any(high > top + kLag || product_exponent(vs_now, high, top) > v_exp + kLag)) {
            const float new_top = fmaxf(top, quads_max(high)), down = top - new_top;
            const float new_exp = fmaxf(fmaxf(__builtin_ceilf(v_exp + down), __builtin_ceilf(quads_max(product_exponent(vs_now, high, new_top)))), kNoExp);
            const float keep_o = __builtin_amdgcn_exp2f(v_exp + down - new_exp);
            sum *= __builtin_amdgcn_exp2f(down);
#pragma unroll
            for (int k = 0; k < kOut; ++k) o[k] *= keep_o;
            top = new_top;
            v_exp = new_exp;
        }
        // weights times the values' scale in one exponential; their sum is divided by it
        v_bad = v_bad || (any && vs_now != vs_now);
        const float lift = any ? scale_log(vs_now, v_exp) : 0.0f, base = (float)kBias - top + lift;
        float w[kMine], run = 0.0f;
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], f, base));
            run += w[e];
        }
        sum = __builtin_fmaf(run, __builtin_amdgcn_exp2f(-lift), sum);
        h8 wh[kMine / 8], wl[PACK ? 1 : kMine / 8];
#pragma unroll
        for (int k = 0; k < kMine / 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h2 hi, lo;
                split_pair(w[8 * k + 2 * e], w[8 * k + 2 * e + 1], &hi, &lo);
                if (PACK) hi = col < 8 ? hi : lo;
                wh[k][2 * e] = hi[0], wh[k][2 * e + 1] = hi[1];
                if (!PACK) wl[k][2 * e] = lo[0], wl[k][2 * e + 1] = lo[1];
            }
        if (F8 && tail) {  // what stands behind the last token may be NaN as a code
            const int left = min(max(q.len - tok0, 0), kMine);
#pragma unroll
            for (int k = 0; k < kOut; ++k) {
                uint32_t* u = reinterpret_cast<uint32_t*>(&vf[k]);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    const int m = min(max(left - 4 * t, 0), 4);
                    u[t] = m == 4 ? u[t] : u[t] & ((1u << (8 * m)) - 1u);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kOut; ++k) {
            const h8 lo = code_oct<F8>(vf[k].x, vf[k].y);
            o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, wh[0], o[k], 0, 0, 0);
            if constexpr (!PACK) o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, wl[0], o[k], 0, 0, 0);
            if constexpr (TOK == 64) {
                const h8 hi = code_oct<F8>(vf[k].z, vf[k].w);
                o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, wh[1], o[k], 0, 0, 0);
                if constexpr (!PACK) o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, wl[1], o[k], 0, 0, 0);
            }
        }
        p = np;
    }
    // the waves' results as one: largest maximum, everything scaled to it
    sum = quads_sum(sum);
    if (quads_max(v_bad ? 1.0f : 0.0f) > 0.0f)
#pragma unroll
        for (int k = 0; k < kOut; ++k) o[k] = (f4)(__builtin_nanf(""));
    if (g == 0) {
        part_m[wave][col] = top;
        part_l[wave][col] = sum;
        part_e[wave][col] = v_exp;
    }
    const bool any_bad = __syncthreads_or(bad) != 0;
    float all_top = kNoMax, all_exp = kNoExp;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all_top = fmaxf(all_top, part_m[k][col]);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all_exp = fmaxf(all_exp, part_e[k][col] + (part_m[k][col] - all_top));
    if (wave == 0 && g == 0) row_e[col] = all_exp;
    // (a wave that has seen nothing has sum 0 and O 0; exp2 of its maximum's distance is 0)
    const float mine = __builtin_amdgcn_exp2f(v_exp + (top - all_top) - all_exp);
#pragma unroll
    for (int k = 0; k < kOut; ++k) {
        f4 y = o[k];
        if (PACK)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += from_other_eight(y[e]);
        if (col < ROWS) *reinterpret_cast<f4*>(&part_o[wave * kPart + col * (DP + 4) + k * 16 + 4 * g]) = y * mine;
    }
    __syncthreads();
    const bool whole = parts == 1;
    const int rows = min(ROWS, n_rows - rt * ROWS), tid = threadIdx.x;
    const float nan = __builtin_nanf("");
    const bool vec = c.dim % 4 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
    auto out_row = [&](int r) {
        const int r_all = rt * ROWS + r;
        return (size_t)(q.r0 + r_all / a.group) * a.n_head + h * a.group + r_all % a.group;
    };
    auto store_out = [&](int r, int d, f4 x) {
        float* y = dst + out_row(r) * c.dim + d;
        if (vec) {
            if (d < c.dim) *reinterpret_cast<f4*>(y) = x;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < c.dim) y[e] = x[e];
        }
    };
    auto lse_of = [&](float l, float m) {
        return l == 0.0f ? -__builtin_inff() : (__builtin_amdgcn_logf(l) + m - (float)kBias) * kLn2;
    };
    float* piece = whole ? nullptr : scratch + (size_t)blockIdx.x * kPieceFloats<DP, ROWS>;
    for (int at = tid; at < rows * kFours; at += kThreads) {
        const int r = at / kFours, d = at % kFours * 4;
        f4 x = f4{0, 0, 0, 0};
        float m = kNoMax, l = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            x += *reinterpret_cast<const f4*>(&part_o[k * kPart + r * (DP + 4) + d]);
            m = fmaxf(m, part_m[k][r]);
        }
#pragma unroll
        for (int k = 0; k < kWaves; ++k) l += part_l[k][r] * __builtin_amdgcn_exp2f(part_m[k][r] - m);
        // (the unit comes last: before it the numbers are of ordinary size, whatever the values are)
        x = x * (l == 0.0f ? 0.0f : 1.0f / l) * __builtin_amdgcn_exp2f(row_e[r]);
        if (any_bad) x = f4{nan, nan, nan, nan}, l = nan;
        if (!whole) {
            *reinterpret_cast<f4*>(piece + r * DP + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(piece + ROWS * DP + 2 * r) = make_float2(m, l * pow2(-kSumDown));
            continue;
        }
        store_out(r, d, x);
        if (lse && d == 0) lse[out_row(r)] = lse_of(l, m);
    }
}

// Joins the pieces of one query row: blockIdx.x counts (sequence, head, row tile), blockIdx.y the row in the tile.
template <int DP, int ROWS>
__global__ __launch_bounds__(256) void join_kernel(Kv8Cache c, Kv8Batch b, Kv8Attn a, float* __restrict__ dst,
                                                   float* __restrict__ lse, const float* __restrict__ scratch, int target,
                                                   int whole_pages, int max_tiles) {
    __shared__ __align__(16) float part[1024 / DP][DP];
    __shared__ float part_m[1024 / DP], part_l[1024 / DP];
    const int rt = blockIdx.x % max_tiles, h = blockIdx.x / max_tiles % c.n_kv, s = blockIdx.x / max_tiles / c.n_kv;
    const int r = blockIdx.y, r_all = rt * ROWS + r;
    const SeqCut cut = find_cut(b, a, c.n_kv, ROWS, target, whole_pages, false, s, 0);
    const Kv8Seq q = cut.q;
    const int parts = cut.parts;
    if (r_all >= q.n * a.group || parts == 1) return;
    const float* first = scratch + (size_t)(cut.first + (h * cut.work.tiles + rt) * parts) * kPieceFloats<DP, ROWS>;
    // four columns to a thread; the threads that share them take every kGroups-th piece, each with its own maximum
    constexpr int kFours = DP / 4, kGroups = 256 / kFours;
    const int d4 = threadIdx.x % kFours, group = threadIdx.x / kFours;
    if (group < kGroups) {
        float m = kNoMax, l = 0.0f;
        f4 x = f4{0, 0, 0, 0};
        constexpr int kAhead = 4;  // pieces asked for at once
        for (int k0 = group; k0 < parts; k0 += kAhead * kGroups) {
            float2 ml[kAhead];
            f4 y[kAhead];
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                const int k = k0 + n * kGroups;
                const float* piece = first + (size_t)min(k, parts - 1) * kPieceFloats<DP, ROWS>;
                ml[n] = *reinterpret_cast<const float2*>(piece + ROWS * DP + 2 * r);
                y[n] = *reinterpret_cast<const f4*>(piece + r * DP + 4 * d4);
                if (k >= parts) ml[n] = make_float2(kNoMax, 0.0f);
            }
            float most = m;
#pragma unroll
            for (int n = 0; n < kAhead; ++n) most = fmaxf(most, ml[n].x);
            const float old = __builtin_amdgcn_exp2f(m - most);
            l *= old;
            x *= old;
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                const float f = ml[n].y * __builtin_amdgcn_exp2f(ml[n].x - most);
                l += f;
                if (k0 + n * kGroups < parts) x += y[n] * f;
            }
            m = most;
        }
        *reinterpret_cast<f4*>(&part[group][4 * d4]) = x;
        if (d4 == 0) {
            part_m[group] = m;
            part_l[group] = l;
        }
    }
    __syncthreads();
    float m = kNoMax, l = 0.0f, y = 0.0f;
    const int d = threadIdx.x;
    if (d >= c.dim) return;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) m = fmaxf(m, part_m[k]);
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const float f = __builtin_amdgcn_exp2f(part_m[k] - m);
        l = __builtin_fmaf(part_l[k], f, l);
        y = __builtin_fmaf(part[k][d], f, y);
    }
    const size_t out = (size_t)(q.r0 + r_all / a.group) * a.n_head + h * a.group + r_all % a.group;
    dst[out * c.dim + d] = l == 0.0f ? 0.0f : y / l;
    if (lse && d == 0) lse[out] = l == 0.0f ? -__builtin_inff() : (__builtin_amdgcn_logf(l) + m - (float)(kBias - kSumDown)) * kLn2;
}

// Query rows of a workgroup: 8 where no sequence has more.
int step_rows(int group, int max_q) { return (int64_t)max_q * group <= 8 ? 8 : kStepRows; }
int max_tiles_of(int group, int max_q) {
    const int rows = step_rows(group, max_q);
    return (int)(((int64_t)max_q * group + rows - 1) / rows);
}

bool takes_gen(const Kv8Attn& a) { return a.softcap > 0.0f || a.window > 0 || a.slopes || a.first || a.prefix; }

// How a call is cut up.
struct StepCut {
    int tiles;     // row tiles of a sequence at most
    int target;    // pieces aimed at
    int whole;     // pages of a sequence that is one piece
    bool join;     // a sequence can have more than one
    bool half;     // waves take half a page at a time
    size_t items;  // upper bound of the pieces
};
// gen: the form with caps and masks by position.
StepCut step_cut(int cus, int dim, bool gen, int window, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    StepCut c;
    c.tiles = max_tiles_of(group, max_q);
    const int64_t tiles = (int64_t)n_seq * n_kv * c.tiles;
    // What runs at a time are two workgroups on a compute unit, one with more than 128 columns: with fewer
    // (sequence, head, row tile)s than that, so many pieces that they are one round together with half a piece each for the
    // rounding up (two sequences of 115000 tokens: 46 us, with half as many again 50). Else they come in rounds, and more of
    // them level out (64 sequences of 500 to 8000 tokens, 8 heads: 72 us, with two thirds of them 74).
    const int64_t slots = dim <= 128 ? 2 * cus : cus;
    c.target = (int)(tiles < slots ? std::max(slots - tiles / 2, slots / 2) : dim <= 128 ? 3 * cus : 2 * cus);
    // Up to which length a sequence stays in one piece: where half the compute units have one already, the pages a wave
    // goes over more cost less than a join (8 heads, whole / cut: 64 sequences of 1000 tokens 27 / 35 us, 32 sequences'
    // drafts over 1024 tokens of 256 columns 33 / 54; but 64 of 500 to 2000 tokens 43 / 39). With fewer it is a join's time
    // against a page's: 12 / 8 pages at 128 columns (one sequence of 700 tokens 10.2 / 10.6 us; 16 sequences of 700
    // 11.9 / 13.5), 8 / 12 with masks (drafts of 16 sequences 19 / 23), 4 / 12 at 256 columns (drafts of 4 sequences
    // 16 / 24 us, one sequence of 700 tokens 12.7 / 15; all with whole pages to a wave).
    c.whole = 2 * tiles > cus ? 24 : dim > 128 ? 4 : gen ? 8 : 12;
    // a window bounds the pages gone over: `window` tokens and one less than the call's rows
    const int64_t most = window > 0 ? std::min<int64_t>(max_pages, ((int64_t)window + max_q + 125) / kPage) : max_pages;
    // (by the table's width: with one of 2048 pages a sequence of 700 tokens pays for an empty join, 13.9 us instead of 10.6)
    c.join = most > c.whole;
    // More than 128 columns leave a compute unit one wave a SIMD, and nothing to do while it waits, unless a wave takes half
    // a page; but that reads V in pieces of 32 bytes, which costs where reading is the bound: half up to 64 pages for a
    // compute unit (256 columns, half / whole pages: drafts of 16 sequences 22.5 / 26.7 us, of 32 26 / 33, one token of 64
    // sequences of 700 43 / 45, of 16 of 500 to 8000 42.4 / 42.9, of 64 of them 152 / 134).
    c.half = dim > 128 && tiles * most <= (int64_t)64 * cus;
    // the total is cut into `target`, and each (sequence, head, row tile) rounds up once
    c.items = std::min((size_t)c.target + (size_t)tiles, (size_t)tiles * (size_t)((max_pages + kStepWaves - 1) / kStepWaves));
    return c;
}
template <int DP, int ROWS>
void launch_step_rows(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch, int cus,
                      hipStream_t stream) {
    const bool gen = takes_gen(a);
    const StepCut cut = step_cut(cus, c.dim, gen, a.window, c.n_kv, a.group, b.n_seq, b.max_q, b.max_pages);
    auto launch = [&](auto tok) {
        constexpr int TOK = decltype(tok)::value;
        auto kernel = c.f8 ? (gen ? step_kernel<DP, ROWS, TOK, true, true> : step_kernel<DP, ROWS, TOK, true, false>)
                           : (gen ? step_kernel<DP, ROWS, TOK, false, true> : step_kernel<DP, ROWS, TOK, false, false>);
        hipLaunchKernelGGL(kernel, dim3((unsigned)cut.items), dim3(64 * kWaves<TOK>), 0, stream, c, b, a, dst, lse, scratch, cut.target,
                           cut.whole);
    };
    bool half = false;
    if constexpr (DP > 128) {
        half = cut.half;
        if (half) launch(std::integral_constant<int, 32>{});
    }
    if (!half) launch(std::integral_constant<int, 64>{});
    if (cut.join)
        hipLaunchKernelGGL((join_kernel<DP, ROWS>), dim3((unsigned)(b.n_seq * c.n_kv * cut.tiles), (unsigned)std::min(ROWS, b.max_q * a.group)),
                           dim3(256), 0, stream, c, b, a, dst, lse, scratch, cut.target, cut.whole, cut.tiles);
}
template <int DP>
void launch_step_dp(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch, int cus,
                    hipStream_t stream) {
    if (step_rows(a.group, b.max_q) == 8) launch_step_rows<DP, 8>(c, b, a, dst, lse, scratch, cus, stream);
    else launch_step_rows<DP, 16>(c, b, a, dst, lse, scratch, cus, stream);
}

}  // namespace

size_t step_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages) {
    // (for the shape alone: what joins most often)
    const StepCut cut = step_cut(cus, dim, true, 0, n_kv, group, n_seq, max_q, max_pages);
    const size_t dp = (size_t)(dim + 63) / 64 * 64;
    return cut.join ? cut.items * (kStepRows * dp + 2 * kStepRows) * sizeof(float) : 0;
}
void launch_attention_step(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, float* scratch,
                           int cus, hipStream_t stream) {
    switch (c.dp) {
    case 64: launch_step_dp<64>(c, b, a, dst, lse, scratch, cus, stream); break;
    case 128: launch_step_dp<128>(c, b, a, dst, lse, scratch, cus, stream); break;
    case 192: launch_step_dp<192>(c, b, a, dst, lse, scratch, cus, stream); break;
    default: launch_step_dp<256>(c, b, a, dst, lse, scratch, cus, stream); break;
    }
}

}  // namespace infr
