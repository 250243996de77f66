// Speculative decoding and windows with vkml::PagedCache on the GPU (links
// libvkml.so). Several sequences, some forks of one another, draft trees, attend
// them in every layer, pick a token after every node (vkml::sample), and keep the
// confirmed path; beside it a second cache gets the confirmed tokens one by one, as
// without drafts. After every step both hold the same keys and values to the bit,
// and each confirmed node's attention is that of the same token there. Then windowed
// attention against a double softmax, and what is refused. Prints a line a case
// ("ok" or what is wrong).
//
// Bounds. Both caches' attention is f32 attention within rounding of the same keys:
// each is off by at most sum p |v| times (2 scale max delta + 2^-22 max|x| + (n / 16 +
// 64) 2^-24 + 2^-20), delta = 2^-22 max|q| sum|k| + (hd + 8) 2^-24 sum|q k|. Here hd
// = 64, n < 400, |k|, |q|, |v| < 6 and |x| < 60: 2 / 8 (2^-22 6 sum|k| + 72 2^-24
// sum|q k|), sum|k| < 64 6 and sum|q k| < 480 (|x| before the scale at most), is less
// than 6.6e-4, so that two outputs are less than 2 6 7e-4 = 8.4e-3 apart: 0.01.
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

constexpr std::int64_t kLayers = 2, kHeads = 8, kKvHeads = 2, kHd = 64, kPage = 16, kPages = 96, kRows = 512, kVocab = 40;
constexpr std::int64_t kLanes = (kHeads + 2 * kKvHeads) * kHd;
constexpr float kNear = 0.01f;

// A token's q | k | v in a layer.
std::vector<float> token_row(std::int64_t token, std::int64_t layer) {
    std::mt19937 gen(static_cast<unsigned>(token * 7 + layer));
    std::normal_distribution<float> d;
    std::vector<float> x(kLanes);
    for (float& y : x) y = std::clamp(d(gen), -4.0f, 4.0f);
    return x;
}

struct Step {
    std::vector<Tensor> out;  // of each layer
};

struct Bench {
    vkml::Context& ctx;
    vkml::PagedCache cache;
    Tensor table;
    RopeStyle style;

    Bench(vkml::Context& c, DType d, RopeStyle s) : ctx(c), cache(c, kLayers, kKvHeads, kHd, kPages, kPage, d), table(vkml::rope_table(c, kRows, kHd, 10000.0f)), style(s) {}

    Step run(const PagedBatch& b, const std::vector<std::int64_t>& tokens, const vkml::PagedTrees* trees) {
        Step s;
        for (std::int64_t layer = 0; layer < kLayers; ++layer) {
            std::vector<float> x;
            for (const std::int64_t t : tokens) {
                const auto r = token_row(t, layer);
                x.insert(x.end(), r.begin(), r.end());
            }
            const Tensor qkv = Tensor::from_data<float>(ctx, x, {static_cast<std::int64_t>(tokens.size()), kLanes});
            const Tensor q = cache.append(layer, b, qkv, table, style, trees);
            s.out.push_back(trees ? cache.attention_tree(layer, b, *trees, q) : cache.attention(layer, b, q));
        }
        return s;
    }

    // A sequence's keys and values of every layer, as stored.
    std::vector<std::byte> stored(std::int64_t id) const {
        std::vector<std::byte> out;
        const auto& row = cache.table().row(id);
        const std::size_t row_bytes = kHd * vkml::element_size(cache.k_pages().dtype());
        for (const Tensor* pool : {&cache.k_pages(), &cache.v_pages()}) {
            const auto bytes = pool->to_bytes();
            for (std::int64_t layer = 0; layer < kLayers; ++layer)
                for (std::int64_t p = 0; p < cache.table().length(id); ++p)
                    for (std::int64_t h = 0; h < kKvHeads; ++h) {
                        const std::int64_t at = ((layer * kPages + row[static_cast<std::size_t>(p / kPage)]) * kKvHeads + h) * kPage + p % kPage;
                        const auto from = bytes.begin() + static_cast<std::ptrdiff_t>(at * static_cast<std::int64_t>(row_bytes));
                        out.insert(out.end(), from, from + static_cast<std::ptrdiff_t>(row_bytes));
                    }
        }
        return out;
    }
};

int speculate(vkml::Context& ctx, DType dtype, RopeStyle style, bool grouped) {
    int wrong = 0;
    std::mt19937 gen(5);
    const auto below = [&](std::int64_t n) { return static_cast<std::int64_t>(gen() % static_cast<unsigned>(n)); };
    Bench with(ctx, dtype, style), without(ctx, dtype, style);
    std::int64_t names = 1000;  // prompt tokens, all different
    std::vector<std::int64_t> a, b, last;  // the sequences in both caches, and each one's last pick
    const auto prompt = [&](std::int64_t n) {
        std::vector<std::int64_t> tokens;
        for (std::int64_t i = 0; i < n; ++i) tokens.push_back(names++);
        a.push_back(with.cache.create());
        b.push_back(without.cache.create());
        with.run(with.cache.batch(std::vector{a.back()}, std::vector{n}), tokens, nullptr);
        without.run(without.cache.batch(std::vector{b.back()}, std::vector{n}), tokens, nullptr);
        last.push_back(below(kVocab));
    };
    prompt(70);
    for (int i = 0; i < 3; ++i) {  // forks of the first, which share its pages
        a.push_back(with.cache.fork(a[0]));
        b.push_back(without.cache.fork(b[0]));
        last.push_back(below(kVocab));
    }
    prompt(5);
    prompt(33);
    for (int step = 0; step < 6; ++step) {
        std::vector<std::int64_t> counts, tokens;
        std::vector<std::int32_t> parents;
        std::vector<std::int32_t> drafted, want;
        for (std::size_t s = 0; s < a.size(); ++s) {
            const std::int64_t n = step == 3 && s == 2 ? 0 : 1 + below(step == 4 ? 40 : 14);
            counts.push_back(n);
            const std::size_t first = drafted.size();
            for (std::int64_t i = 0; i < n; ++i) {
                parents.push_back(i == 0 ? -1 : static_cast<std::int32_t>(below(7) == 0 ? 0 : std::max<std::int64_t>(0, i - 1 - below(3))));
                drafted.push_back(static_cast<std::int32_t>(i == 0 ? last[s] : below(kVocab)));
                want.push_back(static_cast<std::int32_t>(below(kVocab)));
                tokens.push_back(drafted.back());
            }
            for (std::int64_t i = 1; i < n; ++i)  // most nodes' picks are one of their children's tokens
                if (below(4)) want[first + static_cast<std::size_t>(parents[first + static_cast<std::size_t>(i)])] = drafted[first + static_cast<std::size_t>(i)];
        }
        const std::vector<std::int64_t> groups = grouped ? std::vector<std::int64_t>{4} : std::vector<std::int64_t>{};
        const PagedBatch batch = with.cache.batch(a, counts, groups);
        const vkml::PagedTrees trees = with.cache.trees(batch, parents);
        const Step got = with.run(batch, tokens, &trees);
        // logits whose largest is the pick wanted: the draws leave nothing else
        const std::int64_t total = static_cast<std::int64_t>(tokens.size());
        std::vector<float> logits(static_cast<std::size_t>(total * kVocab));
        std::vector<double> draws;
        std::vector<vkml::SamplingOptions> options(static_cast<std::size_t>(total));
        for (std::int64_t t = 0; t < total; ++t) {
            for (std::int64_t i = 0; i < kVocab; ++i) logits[static_cast<std::size_t>(t * kVocab + i)] = i == want[static_cast<std::size_t>(t)] ? 9.0f : static_cast<float>(below(4));
            draws.push_back(static_cast<double>(gen()) / 4294967296.0);
            options[static_cast<std::size_t>(t)].temperature = t % 2 ? 0.8f : 0.0f;
            options[static_cast<std::size_t>(t)].min_p = 0.5f;
        }
        const Tensor picked = vkml::sample(Tensor::from_data<float>(ctx, logits, {total, kVocab}), options, draws);
        if (picked.to_vector<std::int32_t>() != want) std::printf("step %d: the picks are others\n", step), ++wrong;
        const Tensor drafts = Tensor::from_data<std::int32_t>(ctx, drafted, {total});
        const vkml::KeptDrafts kept = with.cache.keep(batch, trees, drafts, picked);
        std::vector<std::vector<float>> rows;
        for (const Tensor& t : got.out) rows.push_back(t.to_vector<float>());
        // the same tokens one at a time in the other cache
        std::size_t first = 0, most = 0;
        for (std::size_t s = 0; s < a.size(); ++s) {
            std::vector<std::int32_t> path;
            if (counts[s] > 0) path.push_back(0);
            while (!path.empty()) {
                std::int32_t next = -1;
                for (std::int32_t i = path.back() + 1; i < counts[s] && next < 0; ++i)
                    if (parents[first + static_cast<std::size_t>(i)] == path.back() && drafted[first + static_cast<std::size_t>(i)] == want[first + static_cast<std::size_t>(path.back())]) next = i;
                if (next < 0) break;
                path.push_back(next);
            }
            most = std::max(most, path.size());
            if (kept.paths[s] != path) std::printf("step %d, sequence %zu: another path\n", step, s), ++wrong;
            const std::int32_t after = path.empty() ? -1 : want[first + static_cast<std::size_t>(path.back())];
            if (kept.next[s] != after) std::printf("step %d, sequence %zu: pick %d for %d\n", step, s, kept.next[s], after), ++wrong;
            for (const std::int32_t node : path) {
                const std::int64_t one = 1;
                const Step ref = without.run(without.cache.batch(std::span(&b[s], 1), std::span(&one, 1)), {drafted[first + static_cast<std::size_t>(node)]}, nullptr);
                for (std::int64_t layer = 0; layer < kLayers; ++layer) {
                    const auto y = ref.out[static_cast<std::size_t>(layer)].to_vector<float>();
                    for (std::size_t i = 0; i < y.size(); ++i) {
                        const float x = rows[static_cast<std::size_t>(layer)][(first + static_cast<std::size_t>(node)) * static_cast<std::size_t>(kHeads * kHd) + i];
                        if (!(std::abs(x - y[i]) <= kNear) && wrong++ < 5) std::printf("step %d, sequence %zu, node %d: %g for %g\n", step, s, node, x, y[i]);
                    }
                }
            }
            if (with.cache.table().length(a[s]) != without.cache.table().length(b[s])) std::printf("step %d, sequence %zu: another length\n", step, s), ++wrong;
            else if (with.stored(a[s]) != without.stored(b[s])) std::printf("step %d, sequence %zu: other keys or values\n", step, s), ++wrong;
            if (after >= 0) last[s] = after;
            first += static_cast<std::size_t>(counts[s]);
        }
        if (most < 2) std::printf("step %d: no draft was kept\n", step), ++wrong;
        if (step == 2) with.cache.compact();
    }
    return wrong;
}

int windows(vkml::Context& ctx, DType dtype) {
    int wrong = 0;
    Bench c(ctx, dtype, RopeStyle::Interleaved);
    const std::vector<std::int64_t> ids = {c.cache.create(), c.cache.create(), c.cache.create()}, counts = {200, 3, 90};
    std::vector<std::int64_t> tokens;
    for (std::int64_t i = 0; i < 293; ++i) tokens.push_back(i);
    c.run(c.cache.batch(ids, counts), tokens, nullptr);
    const PagedBatch batch = c.cache.batch(ids, std::vector<std::int64_t>{1, 2, 40});
    std::vector<float> x;
    for (std::int64_t t = 500; t < 543; ++t) {
        const auto r = token_row(t, 1);
        x.insert(x.end(), r.begin(), r.end());
    }
    const Tensor qkv = Tensor::from_data<float>(ctx, x, {43, kLanes}), q = c.cache.append(1, batch, qkv, Tensor(), RopeStyle::Interleaved);
    const auto qs = q.to_vector<float>();
    for (const auto& [window, sinks] : std::vector<std::pair<std::int64_t, std::int64_t>>{{1, 0}, {20, 4}, {50, 40}, {std::int64_t{1} << 40, 0}, {7, std::int64_t{1} << 40}}) {
        const auto out = c.cache.attention_window(1, batch, q, window, sinks).to_vector<float>();
        std::size_t t = 0;
        for (std::size_t s = 0; s < ids.size(); ++s) {
            const std::int64_t n = c.cache.table().length(ids[s]);
            const auto bytes = c.stored(ids[s]);
            const std::size_t size = vkml::element_size(dtype);
            const auto at = [&](int pool, std::int64_t p, std::int64_t h, std::int64_t d) {
                const std::size_t e = static_cast<std::size_t>((((pool * kLayers + 1) * n + p) * kKvHeads + h) * kHd + d);
                if (size == 4) {
                    float f;
                    std::memcpy(&f, &bytes[e * 4], 4);
                    return static_cast<double>(f);
                }
                std::uint16_t u;
                std::memcpy(&u, &bytes[e * 2], 2);
                const int ex = u >> 10 & 31, m = u & 1023;
                const double v = ex ? std::ldexp(1024 + m, ex - 25) : std::ldexp(m, -24);
                return u & 0x8000 ? -v : v;
            };
            for (std::int64_t i = 0; i < batch.added[s]; ++i, ++t) {
                const std::int64_t pos = batch.before[s] + i;
                for (std::int64_t h = 0; h < kHeads; ++h) {
                    std::vector<double> score;
                    std::vector<std::int64_t> keys;
                    double m = -1e300, sum = 0;
                    for (std::int64_t p = 0; p <= pos; ++p) {
                        if (p <= pos - window && p >= sinks) continue;
                        double y = 0;
                        for (std::int64_t d = 0; d < kHd; ++d) y += static_cast<double>(qs[(t * kHeads + static_cast<std::size_t>(h)) * kHd + static_cast<std::size_t>(d)]) * at(0, p, h / 4, d);
                        score.push_back(y / 8.0);
                        keys.push_back(p);
                        m = std::max(m, score.back());
                    }
                    for (double& y : score) sum += y = std::exp(y - m);
                    for (std::int64_t d = 0; d < kHd; d += 7) {
                        double y = 0;
                        for (std::size_t k = 0; k < keys.size(); ++k) y += score[k] / sum * at(1, keys[k], h / 4, d);
                        const float got = out[(t * kHeads + static_cast<std::size_t>(h)) * kHd + static_cast<std::size_t>(d)];
                        if (!(std::abs(got - y) <= kNear) && wrong++ < 5) std::printf("window %lld, %lld: %g for %g\n", static_cast<long long>(window), static_cast<long long>(sinks), got, y);
                    }
                }
            }
        }
    }
    return wrong;
}

int refusals(vkml::Context& ctx) {
    int wrong = 0;
    const auto throws = [&](const char* what, const auto& f) {
        try {
            f();
        } catch (const vkml::Error& e) {
            if (std::string(e.what()).find(what) != std::string::npos) return;
            std::printf("\"%s\" for \"%s\"\n", e.what(), what), ++wrong;
            return;
        }
        std::printf("no error for \"%s\"\n", what), ++wrong;
    };
    Bench c(ctx, DType::F16, RopeStyle::Interleaved);
    const std::vector<std::int64_t> ids = {c.cache.create(), c.cache.create()};
    const PagedBatch batch = c.cache.batch(ids, std::vector<std::int64_t>{3, 2});
    const std::vector<std::int32_t> fine = {-1, 0, 1, -1, 0};
    const vkml::PagedTrees trees = c.cache.trees(batch, fine);
    throws("parents", [&] { c.cache.trees(batch, std::vector<std::int32_t>{-1, 0}); });
    throws("token 1", [&] { c.cache.trees(batch, std::vector<std::int32_t>{-1, 1, 0, -1, 0}); });
    throws("token 1 of sequence 1", [&] { c.cache.trees(batch, std::vector<std::int32_t>{-1, 0, 0, -1, 2}); });
    throws("token 0", [&] { c.cache.trees(batch, std::vector<std::int32_t>{-2, 0, 0, -1, 0}); });
    const Tensor q = Tensor::zeros(ctx, {5, kHeads, kHd}, DType::F32), ints = Tensor::zeros(ctx, {5}, DType::I32), few = Tensor::zeros(ctx, {4}, DType::I32);
    throws("window", [&] { c.cache.attention_window(0, batch, q, 0); });
    throws("sinks", [&] { c.cache.attention_window(0, batch, q, 5, -1); });
    throws("attention_tree: q", [&] { c.cache.attention_tree(0, batch, trees, Tensor::zeros(ctx, {5, kHeads, 32}, DType::F32)); });
    throws("layer", [&] { c.cache.attention_tree(2, batch, trees, q); });
    throws("drafted and picked", [&] { c.cache.keep(batch, trees, few, ints); });
    throws("drafted and picked", [&] { c.cache.keep(batch, trees, ints, Tensor::zeros(ctx, {5}, DType::F32)); });
    vkml::PagedTrees other;
    throws("another batch", [&] { c.cache.attention_tree(0, batch, other, q); });
    throws("another batch", [&] { c.cache.keep(batch, other, ints, ints); });
    throws("another batch", [&] { c.cache.append(0, batch, Tensor::zeros(ctx, {5, kLanes}, DType::F32), c.table, RopeStyle::Interleaved, &other); });
    const PagedBatch grouped = c.cache.batch(ids, std::vector<std::int64_t>{1, 1}, std::vector<std::int64_t>{2});
    throws("groups", [&] { c.cache.attention_window(0, grouped, Tensor::zeros(ctx, {2, kHeads, kHd}, DType::F32), 5); });
    throws("not as the batch left it", [&] { c.cache.keep(batch, trees, ints, ints); });  // it has grown since
    if (c.cache.table().length(ids[0]) != 4 || c.cache.table().length(ids[1]) != 3) std::printf("a refused call changed a sequence\n"), ++wrong;

    // Rows of a page that a fork reads, or that a page has left, are not moved.
    for (const std::int64_t id : ids) c.cache.release(id);
    const std::int64_t low = c.cache.create(), high = c.cache.create();
    c.cache.batch(std::vector{low}, std::vector<std::int64_t>{1});
    const PagedBatch drafts = c.cache.batch(std::vector{high}, std::vector<std::int64_t>{5});
    const vkml::PagedTrees chain = c.cache.trees(drafts, std::vector<std::int32_t>{-1, 0, 1, 2, 3});
    const std::int64_t fork = c.cache.fork(high);
    throws("another's too", [&] { c.cache.keep(drafts, chain, ints, ints); });
    c.cache.release(fork);
    c.cache.release(low);
    c.cache.compact();
    throws("pages have moved", [&] { c.cache.keep(drafts, chain, ints, ints); });
    if (c.cache.table().length(high) != 5) std::printf("a refused call changed a sequence\n"), ++wrong;
    c.cache.truncate(high, 0);
    const PagedBatch again = c.cache.batch(std::vector{high}, std::vector<std::int64_t>{5});
    c.cache.release(c.cache.fork(high));
    const vkml::KeptDrafts kept = c.cache.keep(again, chain, ints, ints);
    if (kept.paths != std::vector<std::vector<std::int32_t>>{{0, 1, 2, 3, 4}} || c.cache.table().length(high) != 5) std::printf("not kept after a fork that is gone\n"), ++wrong;

    const Tensor logits = Tensor::zeros(ctx, {3, 10}, DType::F32);
    const std::vector<double> u = {0.1, 0.2, 0.3};
    vkml::SamplingOptions o;
    throws("options", [&] { vkml::sample(logits, std::vector<vkml::SamplingOptions>(2), u); });
    throws("random", [&] { vkml::sample(logits, std::vector<vkml::SamplingOptions>(3), std::vector<double>{0.1}); });
    o.temperature = -1.0f;
    throws("temperature", [&] { vkml::sample(logits, std::span(&o, 1), u); });
    o = {}, o.repetition_penalty = 1.5f;
    throws("penalties", [&] { vkml::sample(logits, std::span(&o, 1), u); });
    throws("kernel", [&] { vkml::sample(ints, std::span(&o, 1), u); });
    o = {}, o.temperature = 1.0f;
    if (vkml::sample(logits, std::span(&o, 1), u).to_vector<std::int32_t>() != std::vector<std::int32_t>{1, 2, 3}) std::printf("uniform draws are others\n"), ++wrong;
    if (vkml::sample(Tensor::zeros(ctx, {0, 10}, DType::F32), std::span(&o, 1), {}).numel() != 0) std::printf("no rows\n"), ++wrong;
    return wrong;
}

void report(const std::string& name, int wrong) { std::printf("%s %s\n", wrong ? "WRONG" : "ok", name.c_str()), std::fflush(stdout); }

}  // namespace

int main() {
    vkml::Context ctx;
    int all = 0, w;
    for (const DType d : {DType::F16, DType::F32}) {
        const std::string type = d == DType::F16 ? "f16" : "f32";
        report("drafts " + type, w = speculate(ctx, d, RopeStyle::Interleaved, false)), all += w;
        report("drafts in groups " + type, w = speculate(ctx, d, RopeStyle::RotateHalf, true)), all += w;
        report("windows " + type, w = windows(ctx, d)), all += w;
    }
    report("refusals", w = refusals(ctx)), all += w;
    return all != 0;
}
