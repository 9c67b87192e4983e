// EvictKv8: a sequence's cache cut down to `keep` tokens per KV head, on other pages.
//
// Kept are the first `sink` tokens, the last `recent` and, of those between, the ones with the largest sums of
// attention weight (equal sums: the lower slot), in their order. Two launches:
//   select  one workgroup per (sequence, head): the rank of the smallest kept sum by a radix search, 8 bits a
//           pass over the candidates (LDS counters: integer sums, so the same counts in any order), then the kept
//           slots in ascending order by a running prefix count. Reads 4 bytes a token a pass, from L2 after the
//           first; bound by the passes' latency.
//   move    one workgroup per (new page, head): gathers the kept tokens' codes. A block whose tokens come whole
//           and in place from one block keeps its codes and scale; the others are quantized again from
//           code * scale. Bound by the gather: single bytes of V^T rows and 64-byte pieces of K rows.
#include "kv8.hpp"

namespace infr {

namespace {

constexpr int kSelect = 1024;
constexpr int kMove = 256;

struct EvictSeq {
    int len, n_out;
    bool ok;
};
// Tokens of sequence s before and after, and whether every page either of them needs exists. Uniform over the
// workgroup; `nthreads` threads take part.
__device__ __forceinline__ EvictSeq evict_seq(const Kv8Cache& c, const Kv8Evict& e, int s, int tid, int nthreads) {
    EvictSeq q;
    q.len = e.lens[s];
    const bool fits = q.len >= 0 && (int64_t)q.len <= (int64_t)e.max_pages * kPage;
    q.n_out = fits ? min(q.len, e.keep) : 0;
    bool ok = fits;
    if (fits) {
        for (int p = tid; p * kPage < q.len; p += nthreads) {
            const int page = e.pages[(size_t)s * e.max_pages + p];
            ok = ok && page >= 0 && page < c.n_pages;
        }
        for (int p = tid; p * kPage < q.n_out; p += nthreads) {
            const int page = e.pages_out[(size_t)s * e.out_pages + p];
            ok = ok && page >= 0 && page < c.n_pages;
        }
    }
    q.ok = __syncthreads_and(ok) != 0;
    return q;
}

// Sums as unsigned keys in ascending order; NaN comes last, so that it is kept, and both zeros are one.
__device__ __forceinline__ uint32_t sum_key(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the workgroup's threads and the total; `part` holds one entry per wave.
__device__ __forceinline__ int block_scan(int x, int* part, int* total) {
    const int w = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    const int sum = wave_scan(x);
    __syncthreads();
    if (lane == 63) part[w] = sum;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelect / 64; ++i) {
        if (i < w) before += part[i];
        all += part[i];
    }
    *total = all;
    return before + sum - x;
}

__global__ __launch_bounds__(kSelect) void evict_select_kernel(Kv8Cache c, Kv8Evict e) {
    __shared__ int hist[256];
    __shared__ int part[kSelect / 64];
    __shared__ uint32_t found[2];
    const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
    const EvictSeq q = evict_seq(c, e, s, tid, kSelect);
    int32_t* kept = e.kept + ((size_t)s * c.n_kv + h) * e.keep;
    for (int i = (q.ok ? q.n_out : 0) + tid; i < e.keep; i += kSelect) kept[i] = -1;
    if (h == 0 && tid == 0) e.lens_out[s] = q.ok ? q.n_out : -1;
    if (!q.ok) return;
    if (q.len <= e.keep) {
        for (int i = tid; i < q.len; i += kSelect) kept[i] = i;
        return;
    }
    const int32_t* pages = e.pages + (size_t)s * e.max_pages;
    auto key_at = [&](int j) { return sum_key(c.sums[((size_t)pages[j / kPage] * c.n_kv + h) * kPage + j % kPage]); };
    const int lo = e.sink, hi = q.len - e.recent;  // candidates: more than `need` of them, as len > keep
    int need = e.keep - e.sink - e.recent;
    uint32_t prefix = 0;
    // the need-th largest key, from its top byte down; `need` becomes its rank among the equal ones
    for (int shift = 24; need > 0 && shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelect) hist[i] = 0;
        __syncthreads();
        for (int j = lo + tid; j < hi; j += kSelect) {
            const uint32_t k = key_at(j);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        if (tid < 64) {  // lane l: bins 255 - 4 l downwards
            int mine = 0;
            for (int i = 0; i < 4; ++i) mine += hist[255 - 4 * tid - i];
            const int sum = wave_scan(mine);
            int above = sum - mine;
            if (above < need && need <= sum)
                for (int i = 0; i < 4; ++i) {
                    const int n = hist[255 - 4 * tid - i];
                    if (above < need && need <= above + n) {
                        found[0] = (uint32_t)(255 - 4 * tid - i);
                        found[1] = (uint32_t)(need - above);
                    }
                    above += n;
                }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        need = (int)found[1];
        __syncthreads();
    }
    const bool any = e.keep > e.sink + e.recent;
    int equal_before = 0, out_before = 0;
    for (int base = 0; base < q.len; base += kSelect) {
        const int j = base + tid;
        const bool in = j < q.len, must = in && (j < lo || j >= hi);
        const uint32_t k = in && !must && any ? key_at(j) : 0;
        const bool equal = in && !must && any && k == prefix;
        int total = 0;
        const int rank = equal_before + block_scan(equal ? 1 : 0, part, &total);
        equal_before += total;
        const bool take = must || (in && any && !must && (k > prefix || (equal && rank < need)));
        const int at = out_before + block_scan(take ? 1 : 0, part, &total);
        out_before += total;
        if (take) kept[at] = j;
    }
}

__global__ __launch_bounds__(kMove) void evict_move_kernel(Kv8Cache c, Kv8Evict e) {
    __shared__ uint32_t amax[2][kPage];
    __shared__ uint8_t whole[kPage];
    __shared__ int from[kPage], slot[kPage];
    const int s = blockIdx.z, h = blockIdx.y, po = blockIdx.x, tid = threadIdx.x;
    const int n_out = e.lens_out[s];
    if (n_out <= po * kPage) return;  // also -1: a sequence that was left as it is
    const int cnt = min(kPage, n_out - po * kPage);
    const int to = e.pages_out[(size_t)s * e.out_pages + po];
    const int subs = kPage / c.block;
    const bool f8 = c.f8 != 0;
    const int32_t* kept = e.kept + ((size_t)s * c.n_kv + h) * e.keep + po * kPage;
    if (tid < kPage) {
        const int j = tid < cnt ? kept[tid] : 0;
        from[tid] = e.pages[(size_t)s * e.max_pages + j / kPage];
        slot[tid] = j % kPage;
        const int lead = __shfl(j, tid / c.block * c.block);
        const bool fits = tid >= cnt || (j == lead + tid % c.block && lead % c.block == 0);
        whole[tid] = fits;
        amax[0][tid] = amax[1][tid] = 0;
    }
    __syncthreads();
    const int t = tid >> 2, sub = t / c.block;
    bool copy = true;  // this thread's block comes whole from one block
    for (int o = 0; o < c.block; ++o) copy = copy && whole[sub * c.block + o];
    const bool live = t < cnt;
    const int pg = from[t], sl = slot[t];
    const size_t old_at = ((size_t)pg * c.n_kv + h) * subs + sl / c.block;
    for (int part = 0; part < 2; ++part) {
        const uint8_t* codes = part ? c.v : c.k;
        const float old = (part ? c.vs : c.ks)[old_at];
        auto code_at = [&](int d) { return (uint32_t)codes[part ? v_at(c, pg, h, sl, d) : k_at(c, pg, h, sl, d)]; };
        uint32_t top = 0;
        if (live && !copy)
            for (int d = tid & 3; d < c.dim; d += 4) top = max(top, abs_bits(kv8_value(code_at(d), f8) * old));
        if (top) atomicMax(&amax[part][sub * c.block], top);
        __syncthreads();
        const float scale = copy ? old : kv8_scale(amax[part][sub * c.block], f8);
        if (live && t % c.block == 0 && (tid & 3) == 0) (part ? c.vs : c.ks)[((size_t)to * c.n_kv + h) * subs + sub] = scale;
        for (int d = tid & 3; d < c.dp; d += 4) {
            uint32_t code = 0;
            if (live && d < c.dim) code = copy ? code_at(d) : kv8_code(kv8_value(code_at(d), f8) * old, scale, f8);
            if (live) (part ? c.v : c.k)[part ? v_at(c, to, h, t, d) : k_at(c, to, h, t, d)] = (uint8_t)code;
        }
    }
    if (live && (tid & 3) == 0) {
        const size_t a = ((size_t)pg * c.n_kv + h) * kPage + sl, z = ((size_t)to * c.n_kv + h) * kPage + t;
        c.pos[z] = c.pos[a];
        c.sums[z] = c.sums[a];
    }
}

}  // namespace

void launch_evict_kv8(const Kv8Cache& c, const Kv8Evict& e, hipStream_t stream) {
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)c.n_kv, (unsigned)e.n_seq), dim3(kSelect), 0, stream, c, e);
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)e.out_pages, (unsigned)c.n_kv, (unsigned)e.n_seq), dim3(kMove), 0,
                       stream, c, e);
}

}  // namespace infr
