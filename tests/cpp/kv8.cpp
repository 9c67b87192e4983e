// The 8-bit KV cache through the C++ host side: a prompt and two single tokens in one plan each (write, attention, sums),
// then an eviction. Expected values come from the cache's own codes, decoded here, in double.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <numeric>
#include <random>
#include <vector>

#include "../../include/infr_hip.hpp"

using namespace infr;

static int g_failed = 0;
#define EXPECT(cond, ...)                                     \
    do {                                                      \
        if (!(cond)) {                                        \
            ++g_failed;                                       \
            std::printf("  FAILED %s: ", #cond);              \
            std::printf(__VA_ARGS__);                         \
            std::printf("\n");                                \
        }                                                     \
    } while (0)

static constexpr uint32_t kKv = 2, kHeads = 4, kDim = 64, kPages = 6, kMaxPages = 3;

struct Cached {
    std::vector<double> k, v;  // [len][kDim]
    std::vector<float> sums;
};
// Tokens of KV head h on these pages, decoded from the buffer's bytes (int8, blocks of 16).
static Cached cached(const std::vector<uint8_t>& buf, const Kv8& g, const std::vector<int32_t>& pages, uint32_t len, uint32_t h) {
    const infr_hip_kv8_layout_t l = g.layout();
    Cached c;
    c.k.resize(len * kDim);
    c.v.resize(len * kDim);
    for (uint32_t t = 0; t < len; ++t) {
        const size_t at = (size_t)pages[t / 64] * kKv + h, slot = t % 64;
        float ks, vs, sum;
        std::memcpy(&ks, &buf[l.k_scale + (at * 4 + slot / 16) * 4], 4);
        std::memcpy(&vs, &buf[l.v_scale + (at * 4 + slot / 16) * 4], 4);
        std::memcpy(&sum, &buf[l.sums + (at * 64 + slot) * 4], 4);
        c.sums.push_back(sum);
        for (uint32_t d = 0; d < kDim; ++d) {
            c.k[t * kDim + d] = (double)(int8_t)buf[l.k + at * 64 * kDim + slot * 64 + d] * ks;
            c.v[t * kDim + d] = (double)(int8_t)buf[l.v + (at * kDim + d) * 64 + slot] * vs;
        }
    }
    return c;
}

int main() {
    try {
        HipBackend be(0);
        const Kv8 g{kPages, kKv, kDim, 1};
        const Buffer cache = be.alloc(g.nbytes(), BufferUsage::KvCache);
        std::vector<int32_t> pages = {4, 0, 3};
        std::mt19937 rng(1);
        std::normal_distribution<float> normal;
        auto up = [&](const auto& v) {
            Buffer b = be.alloc(v.size() * 4, BufferUsage::Activations);
            be.upload(b, v);
            return b;
        };
        uint32_t len = 0;
        for (uint32_t n : {100u, 1u, 1u}) {
            len += n;
            const Kv8Batch batch{n, 1, n, kMaxPages};
            Graph graph;
            Bindings binds;
            std::vector<Buffer> held;
            auto tensor = [&](Buffer b, TensorDesc d) {
                const TensorId t = graph.input(std::move(d));
                held.push_back(std::move(b));
                binds.bind(t, held.back());
                return t;
            };
            held.reserve(16);
            std::vector<float> q(n * kHeads * kDim), k(n * kKv * kDim), v(n * kKv * kDim);
            for (auto* x : {&q, &k, &v})
                for (float& y : *x) y = normal(rng);
            std::vector<int32_t> pos(n), start = {0, (int32_t)n}, lens = {(int32_t)len}, slots = {0};
            std::iota(pos.begin(), pos.end(), (int32_t)(len - n));
            const TensorId tq = tensor(up(q), {{n, kHeads * kDim}, DType::F32}), tk = tensor(up(k), {{n, kKv * kDim}, DType::F32});
            const TensorId tv = tensor(up(v), {{n, kKv * kDim}, DType::F32}), tc = graph.input({{g.nbytes()}, DType::I8});
            binds.bind(tc, cache);
            const TensorId tpos = tensor(up(pos), {{n}, DType::I32}), tpages = tensor(up(pages), {{1, kMaxPages}, DType::I32});
            const TensorId tstart = tensor(up(start), {{2}, DType::I32}), tlens = tensor(up(lens), {{1}, DType::I32});
            const TensorId tslots = tensor(up(slots), {{1}, DType::I32});
            const TensorId tdst = tensor(be.alloc(q.size() * 4, BufferUsage::Activations), {{n, kHeads * kDim}, DType::F32});
            const size_t dst_at = held.size() - 1;
            const TensorId tlse = tensor(be.alloc(n * kHeads * 4, BufferUsage::Activations), {{n, kHeads}, DType::F32});
            graph.push(op::WriteKv8{tk, tv, tc, tpos, tpages, tstart, tlens, tslots, g, batch});
            op::AttentionKv8 att{tq, tc, tdst, tpos, tpages, tstart, tlens, g, batch, kHeads};
            att.lse = tlse;
            graph.push(att);
            graph.push(op::ScoreKv8{tq, tc, tlse, tpos, tpages, tstart, tlens, g, batch, kHeads});
            std::vector<uint8_t> before(g.nbytes()), bytes(g.nbytes());
            be.download(cache, before);
            const Plan plan = be.compile(graph);
            be.execute(plan, binds);
            std::vector<float> out(q.size());
            be.download(held[dst_at], out);
            be.download(cache, bytes);
            const float scale = (float)(1.0 / std::sqrt((double)kDim));
            for (uint32_t h = 0; h < kKv; ++h) {
                const Cached c = cached(bytes, g, pages, len, h), old = cached(before, g, pages, len, h);
                for (uint32_t t = 0; t < n; ++t)  // cached values: off by half a code step, and by the scale's own rounding
                    for (uint32_t d = 0; d < kDim; ++d) {
                        float ks;
                        const uint32_t slot = (len - n + t) % 64;
                        std::memcpy(&ks, &bytes[g.layout().k_scale + (((size_t)pages[(len - n + t) / 64] * kKv + h) * 4 + slot / 16) * 4], 4);
                        const double x = k[(t * kKv + h) * kDim + d];
                        EXPECT(std::fabs(c.k[(len - n + t) * kDim + d] - x) <= 0.5001 * ks, "token %u column %u", t, d);
                    }
                std::vector<double> sums(len, 0.0), slack(len, 0.0);
                double vmax = 0;
                for (double x : c.v) vmax = std::max(vmax, std::fabs(x));
                for (uint32_t t = 0; t < n; ++t)
                    for (uint32_t u = h * 2; u < h * 2 + 2; ++u) {
                        const uint32_t see = len - n + t + 1;
                        std::vector<double> s(see);
                        double size = 0, sum = 0;
                        for (uint32_t j = 0; j < see; ++j) {
                            double x = 0, a = 0;
                            for (uint32_t d = 0; d < kDim; ++d) {
                                const double y = (double)q[(t * kHeads + u) * kDim + d] * c.k[j * kDim + d];
                                x += y;
                                a += std::fabs(y);
                            }
                            s[j] = x * scale;
                            size = std::max(size, a * scale);
                        }
                        const double top = *std::max_element(s.begin(), s.end());
                        for (double& x : s) sum += x = std::exp(x - top);
                        // a score is off by its sum's 22-bit operands (2^-21) and 64 f32 additions (64 * 2^-24) of what its
                        // terms add up to, a weight by twice that; the sums over at most 102 tokens by 102 * 2^-24
                        const double off = 2 * size * (std::ldexp(1, -21) + std::ldexp(1, -18)) + std::ldexp(1, -17);
                        for (uint32_t d = 0; d < kDim; ++d) {
                            double y = 0;
                            for (uint32_t j = 0; j < see; ++j) y += s[j] / sum * c.v[j * kDim + d];
                            EXPECT(std::fabs(out[(t * kHeads + u) * kDim + d] - y) <= 2 * off * vmax, "row %u head %u column %u", t, u, d);
                        }
                        for (uint32_t j = 0; j < see; ++j) {
                            sums[j] += s[j] / sum;
                            slack[j] += s[j] / sum * 2 * off;
                        }
                    }
                for (uint32_t j = 0; j < len; ++j) {
                    const double want = (j < len - n ? old.sums[j] : 0.0) + sums[j];
                    EXPECT(std::fabs(c.sums[j] - want) <= slack[j] + want * 2 * n * std::ldexp(1, -24), "sum of token %u: %g, not %g", j, c.sums[j], want);
                }
            }
        }
        // the cache cut down to 40 tokens a head: 2 first, 10 last, the 28 of the largest sums between
        constexpr uint32_t keep = 40, sink = 2, recent = 10;
        std::vector<uint8_t> bytes(g.nbytes());
        be.download(cache, bytes);
        Graph graph;
        Bindings binds;
        const TensorId tc = graph.input({{g.nbytes()}, DType::I8}), tp = graph.input({{1, kMaxPages}, DType::I32});
        const TensorId tl = graph.input({{1}, DType::I32}), to = graph.input({{1, 1}, DType::I32});
        const TensorId tlo = graph.output({{1}, DType::I32}), tk = graph.output({{1, kKv, keep}, DType::I32});
        const Buffer bp = up(pages), bl = up(std::vector<int32_t>{(int32_t)len}), bo = up(std::vector<int32_t>{5});
        const Buffer blo = be.alloc(4, BufferUsage::Readback), bk = be.alloc(kKv * keep * 4, BufferUsage::Readback);
        binds.bind(tc, cache).bind(tp, bp).bind(tl, bl).bind(to, bo).bind(tlo, blo).bind(tk, bk);
        graph.push(op::EvictKv8{tc, tp, tl, to, tlo, tk, g, 1, kMaxPages, keep, sink, recent});
        const Plan plan = be.compile(graph);
        be.execute(plan, binds);
        std::vector<int32_t> lens_out(1), kept(kKv * keep);
        be.download(blo, lens_out);
        be.download(bk, kept);
        EXPECT(lens_out[0] == (int32_t)keep, "length %d", lens_out[0]);
        for (uint32_t h = 0; h < kKv; ++h) {
            const Cached c = cached(bytes, g, pages, len, h);
            std::vector<int32_t> mid(len - sink - recent), want;
            std::iota(mid.begin(), mid.end(), (int32_t)sink);
            std::stable_sort(mid.begin(), mid.end(), [&](int32_t a, int32_t b) { return c.sums[a] > c.sums[b]; });
            mid.resize(keep - sink - recent);
            for (uint32_t i = 0; i < sink; ++i) want.push_back((int32_t)i);
            std::sort(mid.begin(), mid.end());
            want.insert(want.end(), mid.begin(), mid.end());
            for (uint32_t i = len - recent; i < len; ++i) want.push_back((int32_t)i);
            EXPECT(std::equal(want.begin(), want.end(), kept.begin() + h * keep), "head %u keeps other tokens", h);
        }
        // what the kernels do not take is refused when the graph is compiled
        Graph wide;
        const TensorId x = wide.input({{1}, DType::F32});
        wide.push(op::AttentionKv8{x, x, x, x, x, x, x, Kv8{1, 1, 300, 1}, Kv8Batch{1, 1, 1, 1}, 1});
        bool threw = false;
        try {
            const Plan p = be.compile(wide);
        } catch (const Error& e) {
            threw = e.kind == ErrorKind::Unsupported;
        }
        EXPECT(threw, "head_dim 300 was accepted");
    } catch (const Error& e) {
        std::printf("no usable gfx950 device, or a call failed: %s\n", e.what());
        return 99;
    }
    std::printf("%s\n", g_failed ? "FAILED" : "ok");
    return g_failed ? 1 : 0;
}
