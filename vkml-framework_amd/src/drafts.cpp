// drafts.cpp -- vkml::PagedCache's windows and trees of drafted tokens over the C
// ABI (vkml_attend_pages_window, vkml_attend_pages_tree, vkml_keep_drafts).
#include <algorithm>
#include <string>

#include "paged.hpp"

namespace vkml {

using detail::check;
using detail::TensorAccess;
using namespace detail::paged;

Tensor PagedCache::attention_window(std::int64_t layer, const PagedBatch& batch, const Tensor& q, std::int64_t window, std::int64_t sinks, float softcap) const {
    if (window < 1 || sinks < 0) throw Error("PagedCache::attention_window: a window of " + std::to_string(window) + " keys, " + std::to_string(sinks) + " sinks");
    // (no sequence has more keys than a table row holds)
    const std::uint32_t w = u32(std::min(window, kMaxKeys)), first = u32(std::min(sinks, kMaxKeys));
    return attend("PagedCache::attention_window", batch, q, softcap, [&](const vkml_attend_pages_params& p, void* workspace, float* out) {
        return vkml_attend_pages_window(&p, w, first, static_cast<const float*>(q.data()), pool(k_, layer), pool(v_, layer), ints(batch.table), ints(batch.lengths),
                                        ints(batch.starts), workspace, out);
    });
}

PagedTrees PagedCache::trees(const PagedBatch& batch, std::span<const std::int32_t> parents) const {
    if (static_cast<std::int64_t>(parents.size()) != batch.tokens) {
        throw Error("PagedCache::trees: " + std::to_string(parents.size()) + " parents of " + std::to_string(batch.tokens) + " new tokens");
    }
    std::int64_t most = 1;
    for (const std::int64_t n : batch.added) most = std::max(most, n);
    if (most > kMaxNodes) throw Error("PagedCache::trees: a tree of more than 4096 tokens");
    PagedTrees t;
    const std::size_t words = static_cast<std::size_t>(most + 31) / 32;
    std::vector<std::uint32_t> seen(parents.size() * words);
    std::vector<std::int32_t> positions(parents.size()), bits(seen.size());
    std::size_t first = 0;
    for (std::size_t s = 0; s < batch.added.size(); ++s) {
        for (std::size_t i = 0; i < static_cast<std::size_t>(batch.added[s]); ++i) {
            const std::int64_t parent = parents[first + i];
            if (parent < -1 || parent >= static_cast<std::int64_t>(i)) {
                throw Error("PagedCache::trees: token " + std::to_string(i) + " of sequence " + std::to_string(s) + " after token " + std::to_string(parent));
            }
            std::uint32_t* row = seen.data() + (first + i) * words;
            positions[first + i] = static_cast<std::int32_t>(batch.before[s]);
            if (parent >= 0) {
                const std::size_t from = first + static_cast<std::size_t>(parent);
                std::copy_n(seen.data() + from * words, words, row);
                positions[first + i] = positions[from] + 1;
            }
            row[i / 32] |= 1u << (i % 32);
            t.deepest = std::max<std::int64_t>(t.deepest, positions[first + i] + 1);
        }
        first += static_cast<std::size_t>(batch.added[s]);
    }
    for (std::size_t i = 0; i < seen.size(); ++i) bits[i] = static_cast<std::int32_t>(seen[i]);
    detail::Runtime& runtime = TensorAccess::runtime(k_);
    t.before = batch.before;
    t.added = batch.added;
    t.parents = array(runtime, {batch.tokens});
    t.seen = array(runtime, {batch.tokens, static_cast<std::int64_t>(words)});
    t.positions = array(runtime, {batch.tokens});
    upload(t.parents, std::vector<std::int32_t>(parents.begin(), parents.end()), "PagedCache::trees");
    upload(t.seen, bits, "PagedCache::trees");
    upload(t.positions, positions, "PagedCache::trees");
    return t;
}

Tensor PagedCache::attention_tree(std::int64_t layer, const PagedBatch& batch, const PagedTrees& trees, const Tensor& q, float softcap) const {
    if (!trees.fit(batch)) throw Error("PagedCache::attention_tree: the trees are of another batch");
    const Shape& s = trees.seen.shape();
    return attend("PagedCache::attention_tree", batch, q, softcap, [&](const vkml_attend_pages_params& p, void* workspace, float* out) {
        return vkml_attend_pages_tree(&p, u32(s[1]), static_cast<const float*>(q.data()), pool(k_, layer), pool(v_, layer), ints(batch.table), ints(batch.lengths),
                                      ints(batch.starts), batch.groups > 0 ? ints(batch.group_starts) : nullptr,
                                      batch.groups > 0 ? ints(batch.group_keys) : nullptr, static_cast<const std::uint32_t*>(trees.seen.data()), workspace, out);
    });
}

KeptDrafts PagedCache::keep(const PagedBatch& batch, const PagedTrees& trees, const Tensor& drafted, const Tensor& picked) {
    const Shape want = {batch.tokens};
    if (!trees.fit(batch)) throw Error("PagedCache::keep: the trees are of another batch");
    for (const Tensor* t : {&drafted, &picked}) {
        if (t->dtype() != DType::I32 || t->shape() != want) {
            throw Error("PagedCache::keep: drafted and picked must be i32 " + to_string(want) + ", got " + std::string(to_string(t->dtype())) + " " + to_string(t->shape()));
        }
    }
    // (Rows move within the new tokens' pages: they have to be the batch's still, and the
    // sequence's own.)
    auto page = batch.new_pages.begin();
    for (std::size_t i = 0; i < batch.ids.size(); ++i) {
        const std::string id = "PagedCache::keep: sequence " + std::to_string(batch.ids[i]);
        if (table_.changes(batch.ids[i]) != batch.changes[i]) throw Error(id + " is not as the batch left it");
        for (const std::int32_t now : table_.pages_from(batch.ids[i], batch.before[i])) {
            if (page == batch.new_pages.end() || now != *page++) throw Error(id + " is not as the batch left it: its pages have moved");
            if (table_.users(now) != 1) throw Error(id + "'s new keys are another's too");
        }
    }
    KeptDrafts kept;
    kept.paths.resize(batch.ids.size());
    if (batch.seqs == 0) return kept;
    // All memory that the call takes comes before any row moves, that of the cuts among it
    // (a cut that changes nothing makes its room).
    std::vector<std::int32_t> nodes(static_cast<std::size_t>(batch.tokens)), many(batch.ids.size());
    kept.next.resize(batch.ids.size());
    for (std::size_t i = 0; i < batch.ids.size(); ++i) {
        kept.paths[i].reserve(static_cast<std::size_t>(batch.added[i]));
        table_.truncate(batch.ids[i], table_.length(batch.ids[i]));
    }
    detail::Runtime& runtime = TensorAccess::runtime(k_);
    const Tensor path = array(runtime, want), counts = array(runtime, {batch.seqs}), next = array(runtime, {batch.seqs});
    vkml_keep_drafts_params p{};
    p.kv_heads = u32(kv_heads_);
    p.head_dim = u32(head_dim_);
    p.kv_type = detail::type_code(k_.dtype());
    p.page_size = u32(table_.page_size());
    p.pages = u32(table_.pages());
    p.layers = u32(layers_);
    p.seqs = u32(batch.seqs);
    p.tokens = u32(batch.tokens);
    p.table_stride = u32(batch.table.shape().back());
    const auto download = [](std::vector<std::int32_t>& to, const Tensor& from) {
        if (!to.empty()) check(vkml_memcpy_d2h(to.data(), from.data(), to.size() * sizeof(std::int32_t)), "PagedCache::keep");
    };
    try {
        check(vkml_keep_drafts(&p, ints(trees.parents), ints(drafted), ints(picked), ints(batch.table), ints(batch.lengths), ints(batch.starts),
                               static_cast<std::int32_t*>(path.data()), static_cast<std::int32_t*>(counts.data()), static_cast<std::int32_t*>(next.data()), k_.data(),
                               v_.data()),
              "PagedCache::keep");
        download(nodes, path);
        download(many, counts);
        download(kept.next, next);
    } catch (...) {  // rows may have moved, and how is not known
        for (std::size_t i = 0; i < batch.ids.size(); ++i) table_.truncate(batch.ids[i], batch.before[i]);
        throw;
    }
    auto first = nodes.begin();
    for (std::size_t i = 0; i < batch.ids.size(); ++i) {
        kept.paths[i].assign(first, first + many[i]);
        first += static_cast<std::ptrdiff_t>(batch.added[i]);
    }
    for (std::size_t i = 0; i < batch.ids.size(); ++i) table_.truncate(batch.ids[i], batch.before[i] + many[i]);
    return kept;
}

}  // namespace vkml
