// WriteKv8: a call's new key and value rows into the 8-bit cache.
//
// A block of `block` tokens of one head has one scale, so a token that joins an open block can change the codes
// of those before it. The open block's rows are therefore kept in f32 (the tail of the sequence's slot) and the
// block is quantized from them as a whole each time: its codes are those of its tokens taken at once, whatever
// pieces they came in. Tokens of a block whose rows the tail no longer holds (a sequence cut back behind a block
// that had closed, or one that moved to other pages) are taken at their cached values.
//
// One workgroup per (page that gets tokens, head, K or V): 64 tokens x 64 columns at a time, four lanes to a
// token, 16 columns each, so that a token's 64 columns are one 256-byte read and its key codes one 64-byte
// segment; value codes turn in LDS. Bound by HBM on 8 bytes read and 2 written per column of a token; a single
// token per sequence is bound by the launch and four dependent loads (tables, page, tag and tail, codes).
// Measured (8 heads of 128): 8192 tokens of four prompts 17.9 us, 4.6 TB/s read and written (a copy: 5.1); one token
// of each of 64 sequences 8.2 us. (More workgroups on a compute unit by fewer registers spill: 30 us and 18. Codes only
// where a wave has tokens to write: 19.4 us, the branches keep the loads apart.)
#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace infr {

namespace {

constexpr int kThreads = 256;
constexpr int kTurn = kPage + 4;  // LDS row of value codes: 4 bytes of padding keep the columns off one bank

// Pages of a sequence that get tokens.
__device__ __forceinline__ int pages_written(const Kv8Seq& q) {
    return q.ok && q.n > 0 ? (q.len - 1) / kPage - (q.len - q.n) / kPage + 1 : 0;
}

template <int DP, bool F8>
__global__ __launch_bounds__(kThreads) void write_kv8_kernel(Kv8Cache c, Kv8Batch b, const int32_t* __restrict__ slots,
                                                             const float* __restrict__ kx, size_t k_stride,
                                                             const float* __restrict__ vx, size_t v_stride) {
    constexpr int kGroups = DP / 64;
    __shared__ uint32_t amax[kPage];
    __shared__ __align__(16) uint8_t turn[64 * kTurn];
    int rest = 0;
    Kv8Seq q;
    const int s = find_seq(b, (int)blockIdx.x, &rest, &q, [](const Kv8Seq& x) { return pages_written(x); });
    if (s < 0) return;
    const int h = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int slot0 = q.len - q.n;                       // first new token
    const int pi = slot0 / kPage + rest;                 // page of the sequence
    const int page = b.pages[(size_t)s * b.max_pages + pi];
    const int tail_slot = slots[s];
    const bool page_ok = page >= 0 && page < c.n_pages;
    const bool tail_ok = tail_slot >= 0 && tail_slot < c.n_slots;
    const int tid = threadIdx.x, t = tid >> 2, col = (tid & 3) * 16;
    const int subs = kPage / c.block, sub = t / c.block;
    const int tok = pi * kPage + t;                      // token of this thread
    // the block that was open before the call, and what of it the tail holds
    const int open = slot0 / c.block * c.block, have = slot0 - open;
    const float* x = is_v ? vx : kx;
    const size_t stride = is_v ? v_stride : k_stride;
    const size_t tail_at = (((size_t)tail_slot * c.n_kv + h) * 2 + (is_v ? 1 : 0)) * c.block * c.dim;
    int32_t* tag = tail_ok ? c.tag + (((size_t)tail_slot * c.n_kv + h) * 2 + (is_v ? 1 : 0)) * 2 : nullptr;
    const bool raw = rest == 0 && tail_ok && have > 0 && page_ok && tag[0] == page * subs + open % kPage / c.block && tag[1] >= have;
    float* scales = is_v ? c.vs : c.ks;
    const size_t scale_at = ((size_t)page * c.n_kv + h) * subs + sub;
    const bool touched = tok / c.block >= slot0 / c.block && tok / c.block <= (q.len - 1) / c.block;
    const bool is_new = tok >= slot0 && tok < q.len, is_old = touched && tok < slot0;
    const float old_scale = is_old && !raw && page_ok ? scales[scale_at] : 0.0f;

    // this thread's columns, 16 of each 64: zero behind the sequence's end and the row's
    float r[kGroups][16];
    // (the tail's rows are asked for together with the tag that says whether they are the block's)
    const float* src = nullptr;
    if (is_new) src = x + (size_t)(q.r0 + tok - slot0) * stride + (size_t)h * c.dim;
    else if (is_old && tail_ok) src = c.tail + tail_at + (size_t)(tok - open) * c.dim;
    auto load = [&](const float* src) {
        const bool vec = c.dim % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            const int d0 = j * 64 + col;
            if (src && vec && d0 + 16 <= c.dim) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(src + d0 + e);
                    r[j][e] = y.x, r[j][e + 1] = y.y, r[j][e + 2] = y.z, r[j][e + 3] = y.w;
                }
            } else if (src) {
#pragma unroll
                for (int e = 0; e < 16; ++e) r[j][e] = d0 + e < c.dim ? src[d0 + e] : 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) r[j][e] = 0.0f;
            }
        }
    };
    load(src);
    if (is_old && !raw)  // rows the tail does not have: at their values in the cache
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = j * 64 + col + e;
                r[j][e] = 0.0f;
                if (page_ok && d < c.dim) {
                    const size_t at = is_v ? v_at(c, page, h, t, d) : k_at(c, page, h, t, d);
                    r[j][e] = kv8_value<F8>((is_v ? c.v : c.k)[at]) * old_scale;
                }
            }
    // value codes go out in segments: 16 tokens of one column to a thread. Blocks are whole 16s, so a segment is written or
    // left, but for the codes behind the sequence's end in the last one, which are put back as they were.
    const int vd = tid >> 2, vt = (tid & 3) * 16, seg = (pi * kPage + vt) / c.block;
    const int seg_n = seg >= slot0 / c.block ? q.len - pi * kPage - vt : 0;
    uint4 was[kGroups];
    if (is_v && page_ok && seg_n > 0 && seg_n < 16)
#pragma unroll
        for (int j = 0; j < kGroups; ++j) was[j] = *reinterpret_cast<const uint4*>(c.v + v_at(c, page, h, vt, j * 64 + vd));
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, abs_bits(r[j][e]));
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    if ((tid & 3) == 0) amax[t] = top;
    __syncthreads();
    for (int o = 0; o < c.block; ++o) top = max(top, amax[sub * c.block + o]);
    const float scale = kv8_scale(top, F8), inverse = kv8_inverse(scale);
    const Kv8Bounds bounds = kv8_bounds(inverse);
    if (page_ok && touched && t % c.block == 0 && (tid & 3) == 0) scales[scale_at] = scale;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
        if (!page_ok) continue;
        uint32_t w[4], doubt = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = kv8_codes<F8>(&r[j][4 * e], bounds, &doubt);
        if (__any(doubt))
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = kv8_codes_exact<F8>(&r[j][4 * e], scale, inverse);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = inverse == 0.0f ? 0u : w[e];
        if (!is_v) {
            if (is_new || is_old) *reinterpret_cast<uint4*>(c.k + k_at(c, page, h, t, j * 64 + col)) = make_uint4(w[0], w[1], w[2], w[3]);
            continue;
        }
        __syncthreads();  // (page_ok is the workgroup's)
#pragma unroll
        for (int e = 0; e < 16; ++e) turn[(col + e) * kTurn + t] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
        __syncthreads();
        if (seg_n > 0) {
            const uint32_t* src = reinterpret_cast<const uint32_t*>(turn + vd * kTurn + vt);
            uint4 y = make_uint4(src[0], src[1], src[2], src[3]);
            if (seg_n < 16) {
                auto below = [&](int n) { return n >= 4 ? 0xFFFFFFFFu : n > 0 ? (1u << (8 * n)) - 1u : 0u; };
                auto put = [&](uint32_t x, uint32_t old, int n) { return (x & below(n)) | (old & ~below(n)); };
                y = make_uint4(put(y.x, was[j].x, seg_n), put(y.y, was[j].y, seg_n - 4), put(y.z, was[j].z, seg_n - 8),
                               put(y.w, was[j].w, seg_n - 12));
            }
            *reinterpret_cast<uint4*>(c.v + v_at(c, page, h, vt, j * 64 + vd)) = y;
        }
    }
    if (!is_v && page_ok && is_new && (tid & 3) == 0) {
        const size_t at = ((size_t)page * c.n_kv + h) * kPage + t;
        c.pos[at] = b.pos[q.r0 + tok - slot0];
        c.sums[at] = 0.0f;
    }
    // The run's first workgroup, which has read the tail, leaves the rows of the block that is open now in it.
    if (rest != 0 || !tail_ok) return;
    __syncthreads();
    const int last = (q.len - 1) / c.block * c.block;    // first token of that block
    const int lpage = b.pages[(size_t)s * b.max_pages + last / kPage];
    const bool lpage_ok = lpage >= 0 && lpage < c.n_pages;
    int row = tok - last;  // of the tail; this thread's token when its page has the block
    bool put = tok >= last && (is_new || (is_old && !raw && page_ok));  // (rows only the cache had go there at their values)
    if (pi != last / kPage) {
        row = t;
        put = last + t < q.len;
        load(put ? x + (size_t)(q.r0 + last + t - slot0) * stride + (size_t)h * c.dim : nullptr);
    }
    if (put) {
        float* to = c.tail + tail_at + (size_t)row * c.dim;
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            const int d0 = j * 64 + col;
            if (c.dim % 4 == 0 && d0 + 16 <= c.dim) {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(to + d0 + e) = make_float4(r[j][e], r[j][e + 1], r[j][e + 2], r[j][e + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (d0 + e < c.dim) to[d0 + e] = r[j][e];
            }
        }
    }
    if (tid == 0) {
        tag[0] = lpage_ok ? lpage * subs + last % kPage / c.block : -1;
        tag[1] = q.len - last;
    }
}

}  // namespace

void launch_write_kv8(const Kv8Cache& c, const Kv8Batch& b, const int32_t* slots, const float* k, size_t k_stride,
                      const float* v, size_t v_stride, hipStream_t stream) {
    // a run of n rows touches at most n and at most n / 64 + 2 pages
    const unsigned pages = (unsigned)std::min<size_t>((size_t)b.rows, (size_t)b.rows / kPage + 2 * (size_t)b.n_seq);
    auto pick = [&](auto f8) {
        constexpr bool F8 = decltype(f8)::value;
        return c.dp == 64 ? write_kv8_kernel<64, F8> : c.dp == 128 ? write_kv8_kernel<128, F8>
             : c.dp == 192 ? write_kv8_kernel<192, F8> : write_kv8_kernel<256, F8>;
    };
    auto kernel = c.f8 ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(kernel, dim3(pages, (unsigned)c.n_kv, 2), dim3(kThreads), 0, stream, c, b, slots, k, k_stride, v, v_stride);
}

}  // namespace infr
