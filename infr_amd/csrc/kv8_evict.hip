// EvictKv8: a sequence's cache cut down to `keep` tokens per KV head, on other pages.
//
// Kept are the first `sink` tokens, the last `recent` and, of those between, the ones with the largest sums of
// attention weight (equal sums: the lower slot), in their order. Two launches:
//   select  one workgroup per (sequence, head), each thread with a run of neighbouring tokens whose sums stay in its
//           registers: the smallest kept sum is found by counting in 2048 bins over the range of the sums, then over
//           the bin it lies in, 11 bits a pass (integer counts in LDS: the same in any order), until at most 64 are
//           left, which a wave ranks; two prefix sums then give every kept token its place. Bound by the passes' latency.
//   move    one workgroup per (new page, head, K or V): gathers the kept tokens' codes, 16-byte pieces of K rows and
//           single bytes of V^T rows, a lane to a token, so that a wave's bytes lie in as few lines as the tokens'
//           pages allow. A block whose tokens come whole and in place from one block keeps its codes and scale; the
//           others are quantized again from code * scale. Bound by the lines of V that hold any kept token, and by how
//           fast pieces of 64 bytes from all over the cache come in.
// Measured (8 heads of 128): eight sequences of 9000 to 32000 tokens cut to 4096 98.6 us, 28 us select and 70 us move, which
// reads 121 MB and writes 68 (2.7 TB/s; without the gathers of V 34 us less; V's codes through LDS for 8-byte stores, or
// neighbouring new pages on one XCD: no less). Four of 1050 to 1100 tokens cut to 1024: 17.4 us.
#include <type_traits>

#include "kv8.hpp"

namespace infr {

namespace {

typedef short s2 __attribute__((ext_vector_type(2)));

constexpr int kMove = 256;
constexpr int kBinBits = 11, kBins = 1 << kBinBits;

struct EvictSeq {
    int len, n_out;
    bool ok;
};
// Tokens of sequence s before and after, and whether every page either of them needs exists, as far as this thread has
// looked: `nthreads` threads take part.
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
    q.ok = ok;
    return q;
}

// Sums as unsigned keys in ascending order; NaN comes last, so that it is kept, and both zeros are one.
__device__ __forceinline__ uint32_t sum_key(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the workgroup's threads and the total; `part` holds one entry per wave.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* part, int* total) {
    const int w = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    const int sum = wave_scan(x);
    __syncthreads();
    if (lane == 63) part[w] = sum;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
        if (i < w) before += part[i];
        all += part[i];
    }
    *total = all;
    return before + sum - x;
}

// EACH neighbouring tokens of a thread at a time; sequences of more than EACH * THREADS tokens go over them in rounds,
// reading the sums again for each pass.
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS, 4) void evict_select_kernel(Kv8Cache c, Kv8Evict e) {
    __shared__ int part[THREADS / 64];
    __shared__ int hist[kBins];
    __shared__ uint32_t found[3], ends[2], few[64];
    __shared__ int n_few;
    const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
    const EvictSeq q = evict_seq(c, e, s, tid, THREADS);
    const int32_t* pages = e.pages + (size_t)s * e.max_pages;
    const int lo = e.sink, hi = q.len - e.recent;  // candidates: more than `need` of them, as len > keep
    const int need = e.keep - e.sink - e.recent;
    const int span = EACH * THREADS, rounds = (q.len + span - 1) / span;
    // key of each of the thread's tokens, 0 for those that are no candidates: below every number's key
    uint32_t key[EACH];
    auto load = [&](int round) {
        const int j0 = round * span + tid * EACH;
#pragma unroll
        for (int n = 0; n < EACH; n += 4) {
            const int j = j0 + n;  // (four tokens lie in one page)
            float4 x = make_float4(0, 0, 0, 0);
            if (j < q.len) {
                const int page = pages[j / kPage];  // (may be wrong until the check below)
                x = *reinterpret_cast<const float4*>(c.sums + ((size_t)min(max(page, 0), c.n_pages - 1) * c.n_kv + h) * kPage + j % kPage);
            }
            key[n] = j >= lo && j < hi ? sum_key(x.x) : 0;
            key[n + 1] = j + 1 >= lo && j + 1 < hi ? sum_key(x.y) : 0;
            key[n + 2] = j + 2 >= lo && j + 2 < hi ? sum_key(x.z) : 0;
            key[n + 3] = j + 3 >= lo && j + 3 < hi ? sum_key(x.w) : 0;
        }
    };
    const bool fits = q.len >= 0 && (int64_t)q.len <= (int64_t)e.max_pages * kPage;
    if (fits && q.len > e.keep) load(0);
    const bool ok = __syncthreads_and(q.ok) != 0;
    int32_t* kept = e.kept + ((size_t)s * c.n_kv + h) * e.keep;
    for (int i = (ok ? q.n_out : 0) + tid; i < e.keep; i += THREADS) kept[i] = -1;
    if (h == 0 && tid == 0) e.lens_out[s] = ok ? q.n_out : -1;
    if (!ok) return;
    if (q.len <= e.keep) {
        for (int i = tid; i < q.len; i += THREADS) kept[i] = i;
        return;
    }
    // the need-th largest key: `limit`, and how many of those equal to it stay: `ties`
    uint32_t limit = 0;
    int ties = need;
    if (need > 0) {
        uint32_t low = 0xFFFFFFFFu, high = 0;
        for (int r = 0; r < rounds; ++r) {
            if (rounds > 1) load(r);
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                low = key[n] ? min(low, key[n]) : low;
                high = max(high, key[n]);
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            low = min(low, (uint32_t)__shfl_xor((int)low, o));
            high = max(high, (uint32_t)__shfl_xor((int)high, o));
        }
        if (tid < 2) ends[tid] = tid ? 0 : 0xFFFFFFFFu;
        __syncthreads();
        if ((tid & 63) == 0) {
            atomicMin(&ends[0], low);
            atomicMax(&ends[1], high);
        }
        __syncthreads();
        limit = ends[0];
        uint32_t width = ends[1] - ends[0];  // keys in question: limit .. limit + width
        while (width > 0) {
            const int shift = max(32 - __builtin_clz(width) - kBinBits, 0);
            for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
            if (tid == 0) n_few = 0;
            __syncthreads();
            for (int r = 0; r < rounds; ++r) {
                if (rounds > 1) load(r);
#pragma unroll
                for (int n = 0; n < EACH; ++n)
                    if (key[n] && key[n] - limit <= width) atomicAdd(&hist[(key[n] - limit) >> shift], 1);
            }
            __syncthreads();
            // thread i: bins from the top, kBins / THREADS of them
            constexpr int kMine = kBins / THREADS;
            const int top = kBins - 1 - tid * kMine;
            int mine = 0, total = 0;
#pragma unroll
            for (int i = 0; i < kMine; ++i) mine += hist[top - i];
            int above = block_scan<THREADS>(mine, part, &total);
            if (above < ties && ties <= above + mine)
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int n = hist[top - i];
                    if (above < ties && ties <= above + n) {
                        found[0] = (uint32_t)(top - i);
                        found[1] = (uint32_t)(ties - above);
                        found[2] = (uint32_t)n;
                    }
                    above += n;
                }
            __syncthreads();
            const uint32_t base = found[0] << shift, size = (1u << shift) - 1u;
            width = min(size, width - base);
            limit += base;
            ties = (int)found[1];
            const int n_bin = __builtin_amdgcn_readfirstlane((int)found[2]);
            if (width > 0 && n_bin <= 64) {  // few enough for every wave to rank them by itself, a lane to each
                for (int r = 0; r < rounds; ++r) {
                    if (rounds > 1) load(r);
#pragma unroll
                    for (int n = 0; n < EACH; ++n)
                        if (key[n] && key[n] - limit <= width) few[atomicAdd(&n_few, 1)] = key[n];
                }
                __syncthreads();
                const uint32_t mine = (tid & 63) < n_bin ? few[tid & 63] : 0;
                int above = 0, upto = 0;
                for (int i = 0; i < n_bin; ++i) {
                    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
                    above += other > mine ? 1 : 0;
                    upto += other >= mine ? 1 : 0;
                }
                const int l = __builtin_ctzll(__ballot((tid & 63) < n_bin && above < ties && ties <= upto));
                limit = (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
                ties -= __builtin_amdgcn_readlane(above, l);
                width = 0;
            }
            __syncthreads();
        }
    }
    int total = 0;
    int equal_before = 0, out_before = 0;
    for (int r = 0; r < rounds; ++r) {
        if (rounds > 1) load(r);
        const int j0 = r * span + tid * EACH;
        int equal = 0;
#pragma unroll
        for (int n = 0; n < EACH; ++n) equal += need > 0 && key[n] == limit && key[n] ? 1 : 0;
        int rank = equal_before + block_scan<THREADS>(equal, part, &total);
        equal_before += total;
        uint32_t take = 0;
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int j = j0 + n;
            bool yes = j < q.len && (j < lo || j >= hi);
            if (need > 0 && key[n]) {
                if (key[n] > limit) yes = true;
                else if (key[n] == limit) yes = rank++ < ties;
            }
            take |= (uint32_t)yes << n;
        }
        int at = out_before + block_scan<THREADS>(__builtin_popcount(take), part, &total);
        out_before += total;
        for (; take; take &= take - 1) kept[at++] = j0 + __builtin_ctz(take);
    }
}

template <int DP, bool F8>
__global__ __launch_bounds__(kMove) void evict_move_kernel(Kv8Cache c, Kv8Evict e) {
    constexpr int kPieces = DP / 64, kColumns = DP / 4;
    __shared__ uint32_t amax[kPage];
    const int s = blockIdx.z, h = (int)blockIdx.y >> 1, po = blockIdx.x, tid = threadIdx.x;
    const bool is_v = blockIdx.y & 1;
    const int to = e.pages_out[(size_t)s * e.out_pages + po];
    const int subs = kPage / c.block;
    // K: four lanes to a token, 16 columns of each 64; V: a lane to a token, a quarter of the columns to a wave
    const int t = is_v ? tid & 63 : tid >> 2, part = is_v ? tid >> 6 : tid & 3;
    // (kept is -1 behind the last token, and all through for a sequence that was left as it is)
    const int32_t* kept = e.kept + ((size_t)s * c.n_kv + h) * e.keep + po * kPage;
    const int room = min(kPage, e.keep - po * kPage), lead = t / c.block * c.block;
    const int j = t < room ? kept[t] : -1, j0 = lead < room ? kept[lead] : -1;
    const bool live = j >= 0;
    if (tid < kPage) amax[tid] = 0;
    // a tail that holds rows of what was on this page before does not hold those that come now (every workgroup looks at its
    // head's tag of all slots: eight sequences to 4096 tokens take 99 us with 64 slots, 119 with 1024)
    if (kept[0] >= 0)
        for (int i = tid; i < c.n_slots; i += kMove) {
            int32_t* tag = c.tag + (((size_t)i * c.n_kv + h) * 2 + (is_v ? 1 : 0)) * 2;
            const int block = tag[0];
            if (block >= 0 && block / subs == to) tag[0] = -1;
        }
    // amax's top bit marks a block that has to be quantized again
    const bool in_place = !live || (j == j0 + t % c.block && j0 % c.block == 0);
    __syncthreads();
    if (!in_place && part == 0) atomicOr(&amax[t / c.block], 0x80000000u);
    // (a lane without a token reads the first token of page 0 and writes nothing)
    const int page = live ? e.pages[(size_t)s * e.max_pages + j / kPage] : 0, slot = live ? j % kPage : 0;
    const size_t from = (size_t)page * c.n_kv + h, dst = (size_t)to * c.n_kv + h;
    float* scales = is_v ? c.vs : c.ks;
    const float old = scales[from * subs + slot / c.block];
    uint4 kw[kPieces];
    uint32_t vw[kColumns / 4];
    if (!is_v) {
        const uint8_t* src = c.k + from * (DP * kPage) + slot * 64 + part * 16;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) kw[p] = *reinterpret_cast<const uint4*>(src + p * kPage * 64);
    } else {
        const uint8_t* src = c.v + (from * DP + part * kColumns) * kPage + slot;
#pragma unroll
        for (int d = 0; d < kColumns / 4; ++d) {
            vw[d] = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) vw[d] |= (uint32_t)src[(4 * d + n) * kPage] << (8 * n);
        }
    }
    __syncthreads();
    const bool again = amax[t / c.block] >> 31;
    __syncthreads();
    if (again) {
        // the token's code of the largest size, by pairs of 16-bit numbers: every product with the scale is monotone in it
        s2 high = s2{0, 0}, low = s2{0, 0};
        auto look = [&](uint32_t w) {
            if constexpr (F8) {
                high = __builtin_elementwise_max(high, __builtin_bit_cast(s2, w & 0x007F007Fu));
                high = __builtin_elementwise_max(high, __builtin_bit_cast(s2, (w >> 8) & 0x007F007Fu));
            } else {
                const s2 odd = __builtin_bit_cast(s2, w) >> 8, even = __builtin_bit_cast(s2, w << 8) >> 8;
                high = __builtin_elementwise_max(high, __builtin_elementwise_max(odd, even));
                low = __builtin_elementwise_min(low, __builtin_elementwise_min(odd, even));
            }
        };
        if (live && !is_v)
#pragma unroll
            for (int p = 0; p < kPieces; ++p) look(kw[p].x), look(kw[p].y), look(kw[p].z), look(kw[p].w);
        if (live && is_v)
#pragma unroll
            for (int d = 0; d < kColumns / 4; ++d) look(vw[d]);
        const int most = max(max((int)high[0], (int)high[1]), -min((int)low[0], (int)low[1]));
        const float value = F8 ? kv8_value<F8>((uint32_t)most) : (float)most;
        atomicMax(&amax[t / c.block], (live ? abs_bits(value * old) : 0u) | 0x80000000u);
    }
    __syncthreads();
    const float scale = again ? kv8_scale(amax[t / c.block] & 0x7FFFFFFFu, F8) : old, inverse = kv8_inverse(scale);
    const Kv8Bounds bounds = kv8_bounds(inverse);
    auto code = [&](uint32_t w) {
        float x[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) x[n] = kv8_value<F8>((w >> (8 * n)) & 255u) * old;
        uint32_t doubt = 0;
        uint32_t r = kv8_codes<F8>(x, bounds, &doubt);
        if (doubt) r = kv8_codes_exact<F8>(x, scale, inverse);
        return inverse == 0.0f ? 0u : r;
    };
    if (!live) return;
    if (t % c.block == 0 && part == 0) scales[dst * subs + t / c.block] = scale;
    if (!is_v) {
        uint8_t* out = c.k + dst * (DP * kPage) + t * 64 + part * 16;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            if (again) kw[p] = make_uint4(code(kw[p].x), code(kw[p].y), code(kw[p].z), code(kw[p].w));
            *reinterpret_cast<uint4*>(out + p * kPage * 64) = kw[p];
        }
        if (part == 0) {
            c.pos[dst * kPage + t] = c.pos[from * kPage + slot];
            c.sums[dst * kPage + t] = c.sums[from * kPage + slot];
        }
    } else {
        uint8_t* out = c.v + (dst * DP + part * kColumns) * kPage + t;
#pragma unroll
        for (int d = 0; d < kColumns / 4; ++d) {
            const uint32_t w = again ? code(vw[d]) : vw[d];
#pragma unroll
            for (int n = 0; n < 4; ++n) out[(4 * d + n) * kPage] = (uint8_t)(w >> (8 * n));
        }
    }
}

}  // namespace

void launch_evict_kv8(const Kv8Cache& c, const Kv8Evict& e, hipStream_t stream) {
    const dim3 grid((unsigned)c.n_kv, (unsigned)e.n_seq);
    // threads for one round over the sequence where 32 tokens each are enough, no more: they all meet at the barriers (counted by
    // the page table's width: four sequences of 1100 tokens take 27 us with a table of 2048 pages, 17.9 with a tight one)
    const int64_t most = (int64_t)e.max_pages * kPage;
    if (most <= 256 * 8) hipLaunchKernelGGL((evict_select_kernel<256, 8>), grid, dim3(256), 0, stream, c, e);
    else if (most <= 512 * 16) hipLaunchKernelGGL((evict_select_kernel<512, 16>), grid, dim3(512), 0, stream, c, e);
    else hipLaunchKernelGGL((evict_select_kernel<1024, 32>), grid, dim3(1024), 0, stream, c, e);
    auto pick = [&](auto f8) {
        constexpr bool F8 = decltype(f8)::value;
        return c.dp == 64 ? evict_move_kernel<64, F8> : c.dp == 128 ? evict_move_kernel<128, F8>
             : c.dp == 192 ? evict_move_kernel<192, F8> : evict_move_kernel<256, F8>;
    };
    auto move = c.f8 ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(move, dim3((unsigned)e.out_pages, (unsigned)(2 * c.n_kv), (unsigned)e.n_seq), dim3(kMove), 0, stream, c, e);
}

}  // namespace infr
