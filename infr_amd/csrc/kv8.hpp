// The 8-bit KV cache and what its kernels share: geometry, the parts of the cache buffer, the tables
// of a batch, the codes of the two types and the search for the sequence a workgroup works on.
//
// The cache is one buffer of `n_pages` pages of 64 tokens, each for all KV heads. Its parts, each on a
// multiple of 256 bytes, in this order (DP = head_dim rounded up to 64):
//   K codes    u8  [n_pages][n_kv][DP/64][64 tokens][64]   64 bytes of a token side by side: the four lanes
//                                                          that feed a token to the MFMA read one segment
//   V codes    u8  [n_pages][n_kv][DP][64 tokens]          tokens side by side: P.V's MFMA sums over tokens
//   K scales   f32 [n_pages][n_kv][64/block], V scales the same
//   positions  i32 [n_pages][n_kv][64]
//   sums       f32 [n_pages][n_kv][64]                     accumulated attention weight of each token
//   tail       f32 [n_slots][n_kv][2][block][head_dim]     the rows of the block that is open, K then V
//   tag        i32 [n_slots][n_kv][2][2]                   which block of the cache the tail holds, how many rows
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace infr {

constexpr int kPage = 64;
constexpr float kMinScale = 0x1p-96f;

struct Kv8Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    int32_t* pos;
    float* sums;
    float* tail;
    int32_t* tag;
    int32_t n_pages, n_kv, dim, dp, n_slots, block, f8;
};

// The tables that describe a batch, all in device memory.
struct Kv8Batch {
    const int32_t* pos;      // [rows]
    const int32_t* pages;    // [n_seq][max_pages]
    const int32_t* q_start;  // [n_seq + 1]
    const int32_t* lens;     // [n_seq]
    int32_t rows, n_seq, max_q, max_pages;
};

// What AttentionKv8 and ScoreKv8 have in common.
struct Kv8Attn {
    const float* q;
    size_t q_stride;          // floats from row to row
    int32_t n_head, group;    // query heads, and per KV head
    float scale, softcap;     // softcap 0: none
    int32_t window;           // 0: none
    int32_t causal;
    const int32_t* first;     // [rows] or null
    const int32_t* prefix;    // [n_seq] or null
    const float* slopes;      // [n_head] or null
};

struct Kv8Evict {
    const int32_t* pages;
    const int32_t* lens;
    const int32_t* pages_out;  // [n_seq][out_pages]
    int32_t* lens_out;
    int32_t* kept;             // [n_seq][n_kv][keep]
    int32_t n_seq, max_pages, out_pages, keep, sink, recent;
};

void launch_write_kv8(const Kv8Cache& c, const Kv8Batch& b, const int32_t* slots, const float* k, size_t k_stride,
                      const float* v, size_t v_stride, hipStream_t stream);
// f32 scratch an attention launch needs on a device of `cus` compute units, in bytes.
size_t attention_kv8_scratch(int cus, int dim, int n_kv, int group, int n_seq, int max_q, int max_pages);
void launch_attention_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, float* dst, float* lse, void* scratch,
                          int cus, hipStream_t stream);
size_t score_kv8_scratch(int cus, int n_kv, int group, int n_seq, int max_q, int max_pages);
void launch_score_kv8(const Kv8Cache& c, const Kv8Batch& b, const Kv8Attn& a, const float* lse, float decay, void* scratch,
                      int cus, hipStream_t stream);
void launch_evict_kv8(const Kv8Cache& c, const Kv8Evict& e, hipStream_t stream);

#ifdef __HIPCC__
// ---- device side ----

struct Kv8Seq {
    int r0, n, len;  // first row, rows, cached tokens
    bool ok;
};
// Sequence s of the batch. Tables that contradict each other or the shapes give ok = false and, in r0 / n,
// at most max_q rows that lie inside the batch; no other row or page of that sequence is touched.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Batch& b, int s) {
    const int r0 = b.q_start[s], r1 = b.q_start[s + 1], len = b.lens[s];
    Kv8Seq q;
    const int c0 = min(max(r0, 0), b.rows), c1 = min(max(r1, c0), b.rows);
    q.r0 = c0;
    q.n = min(c1 - c0, b.max_q);
    q.len = len;
    q.ok = r0 == c0 && r1 == c1 && c1 - c0 <= b.max_q && len >= q.n && len <= b.max_pages * kPage;
    return q;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// Scale of a block from the largest absolute value's bits, by one multiplication with the reciprocal that is nearest in
// f32; a value that is not finite makes it NaN.
__device__ __forceinline__ float kv8_scale(uint32_t amax_bits, bool f8) {
    if (amax_bits >= 0x7F800000u) return __builtin_nanf("");
    return fmaxf(__builtin_bit_cast(float, amax_bits) * (f8 ? 1.0f / 448.0f : 1.0f / 127.0f), kMinScale);
}
// 1 / scale for kv8_code; 0 for a NaN scale, whose codes are 0.
__device__ __forceinline__ float kv8_inverse(float scale) {
    if (!(scale < __builtin_inff())) return 0.0f;
    const float r = __builtin_amdgcn_rcpf(scale);
    return __builtin_fmaf(__builtin_fmaf(-scale, r, 1.0f), r, r);
}
// Nearest code of x / scale, ties to even. The quotient is the correctly rounded one: x times the inverse, corrected twice
// by its remainder, which a fused multiply-add gives exactly (Markstein's division; scales and codes keep every number in
// it clear of overflow and of what the remainder could lose). It stays below the largest code's rounding border: the scale
// is within 2^-23 of amax / code_max and the quotient is rounded once more.
template <bool F8>
__device__ __forceinline__ uint32_t kv8_code(float x, float scale, float inverse) {
    float y = x * inverse;
    y = __builtin_fmaf(__builtin_fmaf(-scale, y, x), inverse, y);
    y = __builtin_fmaf(__builtin_fmaf(-scale, y, x), inverse, y);
    uint32_t code;
    if constexpr (F8) {
        y = __builtin_copysignf(y, x);  // the remainders of -0 are +0
        code = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xFFu;
    } else code = (uint32_t)(int)fminf(fmaxf(rintf(y), -127.0f), 127.0f) & 0xFFu;
    return inverse == 0.0f ? 0u : code;
}
// Codes without the corrections: the quotient's product with an inverse a little above and with one a little below it. The
// inverse is within 2^-23 of 1 / scale and the correctly rounded quotient within 2^-24 of the true one, so with 2^-22 to
// either side the two products enclose it; rounding is monotone, so where both give one code it is the quotient's. Where
// they do not, `doubt` says so (about one code in 10^5) and kv8_code decides.
struct Kv8Bounds {
    float lo, hi;
};
__device__ __forceinline__ Kv8Bounds kv8_bounds(float inverse) { return {inverse * (1.0f - 0x1p-22f), inverse * (1.0f + 0x1p-22f)}; }
// Four codes side by side. The int8 codes come out of one fused multiply-add each: added to 1.5 * 2^23 a product is rounded
// to whole numbers, ties to even, and stands in the sum's low bits.
template <bool F8>
__device__ __forceinline__ uint32_t kv8_codes(const float* x, Kv8Bounds inv, uint32_t* doubt) {
    if constexpr (F8) {
        int a = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv.lo, x[1] * inv.lo, 0, false);
        a = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv.lo, x[3] * inv.lo, a, true);
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv.hi, x[1] * inv.hi, 0, false);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv.hi, x[3] * inv.hi, b, true);
        *doubt |= (uint32_t)(a ^ b);
        return (uint32_t)a;
    } else {
        uint32_t a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = __builtin_bit_cast(uint32_t, __builtin_fmaf(x[e], inv.lo, 12582912.0f));
            *doubt |= a[e] ^ __builtin_bit_cast(uint32_t, __builtin_fmaf(x[e], inv.hi, 12582912.0f));
        }
        return __builtin_amdgcn_perm(a[1], a[0], 0x0C0C0400u) | __builtin_amdgcn_perm(a[3], a[2], 0x04000C0Cu);
    }
}
// The same in doubt.
template <bool F8>
__device__ __forceinline__ uint32_t kv8_codes_exact(const float* x, float scale, float inverse) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= kv8_code<F8>(x[e], scale, inverse) << (8 * e);
    return w;
}
template <bool F8>
__device__ __forceinline__ float kv8_value(uint32_t code) {
    if constexpr (F8) return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
    else return (float)(int)(int8_t)code;
}

// Byte offset of key code d of token t of (page, head) / of value code d.
__device__ __forceinline__ size_t k_at(const Kv8Cache& c, int page, int h, int t, int d) {
    return ((((size_t)page * c.n_kv + h) * (c.dp / 64) + d / 64) * kPage + t) * 64 + d % 64;
}
__device__ __forceinline__ size_t v_at(const Kv8Cache& c, int page, int h, int t, int d) {
    return (((size_t)page * c.n_kv + h) * c.dp + d) * kPage + t;
}

// Inclusive prefix sum over the 64 lanes of a wave: within rows of 16 lanes, then from row to row, by DPP moves (a
// shuffle through LDS takes ten times as long, and these sums stand before everything else a kernel does).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int x) {
    x += dpp_or_zero<0x111, 0xF>(x);  // one lane up, then 2, 4, 8
    x += dpp_or_zero<0x112, 0xF>(x);
    x += dpp_or_zero<0x114, 0xF>(x);
    x += dpp_or_zero<0x118, 0xF>(x);
    x += dpp_or_zero<0x142, 0xA>(x);  // the sum of row 0 to row 1, of 2 to 3
    x += dpp_or_zero<0x143, 0xC>(x);  // of rows 0 and 1 to 2 and 3
    return x;
}
// Sum over the wave, in the same order of additions everywhere.
__device__ __forceinline__ float wave_total(float x) {
    auto step = [&](int y) { x += __builtin_bit_cast(float, y); };
    step(dpp_or_zero<0x111, 0xF>(__builtin_bit_cast(int, x)));
    step(dpp_or_zero<0x112, 0xF>(__builtin_bit_cast(int, x)));
    step(dpp_or_zero<0x114, 0xF>(__builtin_bit_cast(int, x)));
    step(dpp_or_zero<0x118, 0xF>(__builtin_bit_cast(int, x)));
    step(dpp_or_zero<0x142, 0xA>(__builtin_bit_cast(int, x)));
    step(dpp_or_zero<0x143, 0xC>(__builtin_bit_cast(int, x)));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The sequence that work item `idx` belongs to, where a sequence has count(its tables) >= 0 of them; in *rest the item's
// number within the sequence and in *q its tables; -1 when there are fewer items. Every lane of the wave calls it with
// the same idx: lanes look at 64 sequences at once and pass on the one found.
template <typename F>
__device__ __forceinline__ int find_seq(const Kv8Batch& b, int idx, int* rest, Kv8Seq* q, F count) {
    const int lane = (int)(threadIdx.x & 63);
    for (int base = 0; base < b.n_seq; base += 64) {
        Kv8Seq mine{};
        if (base + lane < b.n_seq) mine = kv8_seq(b, base + lane);
        const int n = base + lane < b.n_seq ? count(mine) : 0;
        const int sum = wave_scan(n);
        const unsigned long long hit = __ballot(idx < sum);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            *rest = idx - (of(sum) - of(n));
            q->r0 = of(mine.r0);
            q->n = of(mine.n);
            q->len = of(mine.len);
            q->ok = of((int)mine.ok) != 0;
            return base + l;
        }
        idx -= __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}
#endif  // __HIPCC__

}  // namespace infr
