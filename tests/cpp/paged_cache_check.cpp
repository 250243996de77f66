// vkml::PagedCache on the GPU (links libvkml.so): prompts, forks, decoding in
// groups, ragged steps, truncation, compaction and a full pool, over two
// layers. After every step each sequence's keys and values are read back
// through its pages and compared with the rotated and rounded inputs, and
// each new token's attention with a double softmax over those stored keys.
// Prints a line a case ("ok" or what is wrong).
//
// Bounds. Stored values: the rotation's two products and a sum, 2^-23
// (|a| + |b|), then f16's half step, 2^-11 of the value (2^-25 below its
// smallest normal number). Attention, with n keys, delta = 2^-22 max|q| sum|k|
// + (hd + 8) 2^-24 sum|q k| a score's error before the scale: sum p |v| times
// (2 scale max delta + 2^-22 max|x| + (n / 16 + 64) 2^-24 + 2^-20).
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <map>
#include <random>
#include <string>
#include <vector>

#include "vkml/vkml.hpp"

namespace {

using vkml::DType;
using vkml::PagedBatch;
using vkml::RopeStyle;
using vkml::Tensor;

constexpr std::int64_t kLayers = 2, kHeads = 8, kKvHeads = 2, kPage = 16, kPages = 24, kRows = 128;
constexpr std::int64_t kLanes = kHeads + 2 * kKvHeads;

struct Case {
    vkml::Context& ctx;
    std::int64_t hd;
    DType dtype;
    RopeStyle style;
    std::int64_t rotary;
    float softcap;
    vkml::PagedCache cache;
    Tensor table;
    std::vector<float> angles;
    std::mt19937 gen{11};
    // The tokens of each sequence: for each layer, its q | k | v.
    using Token = std::vector<std::vector<float>>;
    std::map<std::int64_t, std::vector<Token>> history;
    int wrong = 0;

    Case(vkml::Context& c, std::int64_t head_dim, DType d, RopeStyle s, std::int64_t rotary_dim, float cap)
        : ctx(c), hd(head_dim), dtype(d), style(s), rotary(rotary_dim), softcap(cap), cache(c, kLayers, kKvHeads, head_dim, kPages, kPage, d) {
        if (rotary > 0) {
            table = vkml::rope_table(ctx, kRows, rotary, 10000.0f, vkml::RopeScaling{8.0f, 1.0f, 4.0f, 32});
            angles = table.to_vector<float>();
        }
    }

    // One head's values, turned; `loss` gets the rounding error that they may have.
    std::vector<double> turned(const float* x, std::int64_t at, std::vector<double>& loss) const {
        std::vector<double> y(x, x + hd);
        loss.assign(static_cast<std::size_t>(hd), 0.0);
        for (std::int64_t i = 0; i < rotary / 2; ++i) {
            const std::int64_t a = style == RopeStyle::Interleaved ? 2 * i : i, b = style == RopeStyle::Interleaved ? 2 * i + 1 : i + rotary / 2;
            const double c = angles[static_cast<std::size_t>(at * rotary + 2 * i)], s = angles[static_cast<std::size_t>(at * rotary + 2 * i + 1)];
            y[a] = x[a] * c - x[b] * s;
            y[b] = x[a] * s + x[b] * c;
            loss[a] = 0x1p-23 * (std::abs(x[a] * c) + std::abs(x[b] * s));
            loss[b] = 0x1p-23 * (std::abs(x[a] * s) + std::abs(x[b] * c));
        }
        return y;
    }

    void differs(const char* what, double got, double want, double bound) {
        if (std::abs(got - want) <= bound * 1.001) return;
        if (wrong++ < 5) std::printf("%s: %.9g, not %.9g within %.3g\n", what, got, want, bound);
    }

    void step(const std::vector<std::int64_t>& ids, const std::vector<std::int64_t>& counts, const std::vector<std::int64_t>& groups = {}) {
        const PagedBatch batch = cache.batch(ids, counts, groups);
        std::normal_distribution<float> normal;
        for (std::size_t i = 0; i < ids.size(); ++i)
            for (std::int64_t n = 0; n < counts[i]; ++n) {
                Token token(kLayers);
                for (auto& layer : token)
                    for (std::int64_t j = 0; j < kLanes * hd; ++j) layer.push_back(normal(gen));
                history[ids[i]].push_back(token);
            }
        for (std::int64_t layer = 0; layer < kLayers; ++layer) {
            std::vector<float> rows;
            for (std::size_t i = 0; i < ids.size(); ++i) {
                const auto& h = history[ids[i]];
                for (std::size_t t = h.size() - static_cast<std::size_t>(counts[i]); t < h.size(); ++t)
                    rows.insert(rows.end(), h[t][layer].begin(), h[t][layer].end());
            }
            const Tensor q = cache.append(layer, batch, Tensor::from_data<float>(ctx, rows, {batch.tokens, kLanes * hd}), table, style);
            verify(layer, ids, counts, q, cache.attention(layer, batch, q, softcap));
        }
    }

    void verify(std::int64_t layer, const std::vector<std::int64_t>& ids, const std::vector<std::int64_t>& counts, const Tensor& q, const Tensor& out) {
        const std::vector<float> gq = q.to_vector<float>(), go = out.to_vector<float>();
        const std::vector<float> gk = vkml::cast(cache.k_pages(), DType::F32).to_vector<float>(), gv = vkml::cast(cache.v_pages(), DType::F32).to_vector<float>();
        const double half = dtype == DType::F16 ? 0x1p-11 : 0.0, least = dtype == DType::F16 ? 0x1p-25 : 0.0;
        std::vector<double> loss;
        std::int64_t row = 0;
        for (std::size_t s = 0; s < ids.size(); ++s) {
            const auto& h = history[ids[s]];
            const auto& pages = cache.table().row(ids[s]);
            const auto n = static_cast<std::int64_t>(h.size());
            const auto at = [&](std::int64_t head, std::int64_t p) {
                return (((layer * kPages + pages[static_cast<std::size_t>(p / kPage)]) * kKvHeads + head) * kPage + p % kPage) * hd;
            };
            for (std::int64_t p = 0; p < n; ++p)
                for (std::int64_t head = 0; head < kKvHeads; ++head) {
                    const float* x = h[static_cast<std::size_t>(p)][layer].data();
                    const std::vector<double> k = turned(x + (kHeads + head) * hd, p, loss);
                    for (std::int64_t d = 0; d < hd; ++d) {
                        const double v = x[(kHeads + kKvHeads + head) * hd + d];
                        differs("k", gk[at(head, p) + d], k[d], loss[d] + std::max(half * std::abs(k[d]), least));
                        differs("v", gv[at(head, p) + d], v, std::max(half * std::abs(v), least));
                    }
                }
            const double scale = 1.0 / std::sqrt(static_cast<double>(hd));
            for (std::int64_t t = n - counts[s]; t < n; ++t, ++row)
                for (std::int64_t head = 0; head < kHeads; ++head) {
                    const float* mine = &gq[static_cast<std::size_t>((row * kHeads + head) * hd)];
                    const std::vector<double> want_q = turned(h[static_cast<std::size_t>(t)][layer].data() + head * hd, t, loss);
                    for (std::int64_t d = 0; d < hd; ++d) differs("q", mine[d], want_q[d], loss[d]);
                    double widest = 0.0, top = -INFINITY, off = 0.0, far = 0.0, sum = 0.0;
                    for (std::int64_t d = 0; d < hd; ++d) widest = std::max(widest, std::abs(static_cast<double>(mine[d])));
                    std::vector<double> x;
                    const std::int64_t kv = head / (kHeads / kKvHeads);
                    for (std::int64_t p = 0; p <= t; ++p) {
                        double dot = 0.0, size = 0.0, each = 0.0;
                        for (std::int64_t d = 0; d < hd; ++d) {
                            const double k = gk[at(kv, p) + d];
                            dot += mine[d] * k;
                            size += std::abs(k);
                            each += std::abs(mine[d] * k);
                        }
                        const double score = dot * scale;
                        x.push_back(softcap > 0.0f ? softcap * std::tanh(score / softcap) : score);
                        top = std::max(top, x.back());
                        far = std::max(far, std::abs(score));
                        off = std::max(off, scale * (0x1p-22 * widest * size + static_cast<double>(hd + 8) * 0x1p-24 * each) + softcap * 0x1p-20);
                    }
                    for (double& e : x) sum += e = std::exp(e - top);
                    const double rel = 2 * off + 0x1p-22 * far + (static_cast<double>(t + 1) / 16 + 64) * 0x1p-24 + 0x1p-20;
                    for (std::int64_t d = 0; d < hd; ++d) {
                        double value = 0.0, size = 0.0;
                        for (std::int64_t p = 0; p <= t; ++p) {
                            value += x[static_cast<std::size_t>(p)] * gv[at(kv, p) + d];
                            size += std::abs(x[static_cast<std::size_t>(p)] * gv[at(kv, p) + d]);
                        }
                        differs("out", go[static_cast<std::size_t>((row * kHeads + head) * hd + d)], value / sum, size / sum * rel);
                    }
                }
        }
    }

    std::int64_t fork(std::int64_t id) {
        const std::int64_t copy = cache.fork(id);
        history[copy] = history[id];
        return copy;
    }

    void run() {
        const std::int64_t a = cache.create();
        step({a}, {37});
        const std::int64_t b = fork(a), c = fork(a);  // three pages shared, the last of five keys
        step({a, b, c}, {1, 1, 1}, {3});
        for (int i = 0; i < 14; ++i) step({a, b, c}, {1, 1, 1}, {3});
        const std::int64_t d = cache.create();
        step({c, a, d, b}, {1, 5, 21, 0}, {2});        // a prompt beside decoding, one sequence idle
        cache.release(a);
        history.erase(a);
        cache.truncate(b, 40);                          // into a page of its own
        history[b].resize(40);
        cache.truncate(c, 20);                          // into one that b holds too
        history[c].resize(20);
        cache.compact();
        step({b, c, d}, {1, 1, 1}, {2, 1});
        step({b, c, d}, {2, 30, 1}, {2});
        const std::vector<std::int32_t> before = cache.table().row(d);
        bool refused = false;
        try {
            step({d}, {16 * kPages});
        } catch (const vkml::Error&) {
            refused = cache.table().row(d) == before;
        }
        if (!refused) ++wrong, std::printf("a full pool was not refused\n");
        step({d}, {1});
        step({}, {});
    }
};

int refusals(vkml::Context& ctx) {
    int wrong = 0;
    const auto refused = [&](const char* why, const auto& call) {
        try {
            call();
        } catch (const vkml::Error& e) {
            if (std::string(e.what()).find(why) != std::string::npos) return;
            std::printf("refused with: %s\n", e.what());
        }
        ++wrong;
        std::printf("not refused: %s\n", why);
    };
    refused("no kernel", [&] { vkml::PagedCache(ctx, 1, 2, 64, 4, 16, DType::BF16); });
    refused("power of two", [&] { vkml::PagedCache(ctx, 1, 2, 64, 4, 24, DType::F16); });
    refused("layers", [&] { vkml::PagedCache(ctx, 0, 2, 64, 4, 16, DType::F16); });
    vkml::PagedCache cache(ctx, 1, 2, 64, 4, 16, DType::F16);
    const std::vector<std::int64_t> ids = {cache.create()}, one = {1}, two = {2}, none = {};
    refused("a group of 2", [&] { cache.batch(ids, one, two); });
    refused("counts", [&] { cache.batch(ids, none); });
    if (cache.table().length(ids[0]) != 0) ++wrong;
    const PagedBatch batch = cache.batch(ids, one);
    const Tensor qkv = Tensor::zeros(ctx, {1, 8 * 64}, DType::F32), q = Tensor::zeros(ctx, {1, 4, 64}, DType::F32);
    refused("no layer 1", [&] { cache.append(1, batch, qkv, Tensor(), RopeStyle::Interleaved); });
    refused("qkv must be", [&] { cache.append(0, batch, q, Tensor(), RopeStyle::Interleaved); });
    refused("qkv must be", [&] { cache.append(0, batch, Tensor::zeros(ctx, {2, 8 * 64}, DType::F32), Tensor(), RopeStyle::Interleaved); });
    refused("qkv must be", [&] { cache.append(0, batch, Tensor::zeros(ctx, {1, 4 * 64}, DType::F32), Tensor(), RopeStyle::Interleaved); });
    refused("rope_table", [&] { cache.append(0, batch, qkv, vkml::rope_table(ctx, 8, 128, 1e4f), RopeStyle::Interleaved); });
    refused("no layer -1", [&] { cache.attention(-1, batch, q); });
    refused("q must be", [&] { cache.attention(0, batch, Tensor::zeros(ctx, {1, 3, 64}, DType::F32)); });
    refused("q must be", [&] { cache.attention(0, batch, Tensor::zeros(ctx, {2, 4, 64}, DType::F32)); });
    refused("softcap", [&] { cache.attention(0, batch, q, -1.0f); });
    return wrong;
}

}  // namespace

int main() {
    vkml::Context ctx;
    int wrong = refusals(ctx);
    std::printf("%s refusals\n", wrong ? "WRONG" : "ok");
    for (const std::int64_t hd : {64, 128})
        for (const DType dtype : {DType::F16, DType::F32})
            for (const RopeStyle style : {RopeStyle::Interleaved, RopeStyle::RotateHalf}) {
                const bool half = style == RopeStyle::RotateHalf;
                Case c(ctx, hd, dtype, style, hd == 64 && half ? 0 : half ? hd / 2 : hd, dtype == DType::F32 && half ? 5.0f : 0.0f);
                c.run();
                std::printf("%s head_dim=%lld %s rotary=%lld softcap=%g\n", c.wrong ? "WRONG" : "ok", static_cast<long long>(hd),
                            std::string(to_string(dtype)).c_str(), static_cast<long long>(c.rotary), c.softcap);
                std::fflush(stdout);
                wrong += c.wrong;
            }
    return wrong ? 1 : 0;
}
